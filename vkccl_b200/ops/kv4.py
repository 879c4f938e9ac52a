# SPDX-License-Identifier: Apache-2.0
"""A paged key/value cache held in 4 bits, and attention over it.

kv4_alloc(pages, page_size, kv_heads, head_dim)   the cache of one layer
kv4_append(cache, k, v, slots)                    writes keys and values
kv4_append_rope(cache, q, k, v, slots, ...)       the same after norm and rotation, in one launch
kv4_read(cache, slots)                            the values that it holds
kv4_attention(q, cache, block_table, kv_lens, q_starts)
                                                  causal attention of ragged query rows
kv4_attention_status()                            whether an attention launch gave up

64 channels of a token share a bf16 scale and midpoint: value = midpoint +
scale * (code - 7.5), 4.5 bits a value.  Slots, tables and lengths are those
of ``vkccl_b200.ops.paging.plan_pages``.  All calls are stream-ordered on
torch's current stream, allocate through torch and may be captured into CUDA
graphs.  They are for serving: there are no gradients, and outputs have no
autograd history.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from vkccl_b200._lib import lib
from vkccl_b200.comm import _check
from vkccl_b200.ops._args import DTYPES, cache4, call, current_device, float16s, fresh, heads, on_device, rope_of, vector

MAX_BATCH = 4096


def kv4_alloc(pages: int, page_size: int, kv_heads: int, head_dim: int, device="cuda") -> torch.Tensor:
    """uint8 [pages, kv heads, page_size / 16, 18 * head_dim]; page_size a multiple of 16, head_dim 64 or 128."""
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
    if page_size < 16 or page_size % 16:
        raise ValueError(f"page_size must be a multiple of 16, got {page_size}")
    if pages < 1 or kv_heads < 1 or pages * page_size > 2**31 - 1:
        raise ValueError("pages and kv_heads must be positive, and pages * page_size fit in 31 bits")
    return torch.zeros((pages, kv_heads, page_size // 16, 18 * head_dim), dtype=torch.uint8, device=device)


def kv4_append(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Writes k, v [T, kv heads, D] (bf16 or fp16) to slots [T] (int32).

    A negative slot, or one behind the cache, is skipped; the others must be
    distinct.  A group of 64 channels with a NaN or an infinity (or whose
    extremes' sum or difference is not an f32) reads back as NaN.
    """
    dev, dtype = float16s(k, "k"), k.dtype
    t, _, dim = k.shape
    c, n, _, _ = cache4(cache, dim, dev)
    hk, hv = heads(k, "k", dtype, dev, t, dim, n), heads(v, "v", dtype, dev, t, dim, n)
    at = vector(slots, "slots", torch.int32, t, dev)
    call(lib().vcclKv4Append, "vcclKv4Append", dev, c, hk, hv, at, None, None, None, t, DTYPES[dtype])


def kv4_append_rope(cache: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
                    positions: torch.Tensor, inv_freq: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                    k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                    q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``qk_norm_rope`` of q and k, and ``kv4_append`` of the result and v, in one launch: the same bits.  Returns q_out."""
    dev, dtype = float16s(q, "q"), q.dtype
    t, nq, dim = q.shape
    c, n, _, _ = cache4(cache, dim, dev)
    hq = heads(q, "q", dtype, dev, t, dim)
    hk, hv = heads(k, "k", dtype, dev, t, dim, n), heads(v, "v", dtype, dev, t, dim, n)
    at = vector(slots, "slots", torch.int32, t, dev)
    rope = rope_of(positions, inv_freq, q_weight, k_weight, eps, interleaved, dtype, dev, t, dim)
    if q_out is None:
        q_out, oq = fresh(q, t, nq, dim)
    else:
        oq = heads(q_out, "q_out", dtype, dev, t, dim, nq, True)
    call(lib().vcclKv4Append, "vcclKv4Append", dev, c, hk, hv, at, rope, hq, oq, t, DTYPES[dtype])
    return q_out


def kv4_read(cache: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
             k_out: Optional[torch.Tensor] = None, v_out: Optional[torch.Tensor] = None
             ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values [T, kv heads, D] that the cache holds at slots [T]; zero where a slot is skipped."""
    if dtype not in DTYPES:
        raise ValueError("dtype must be bf16, fp16 or f32")
    c, n, dim, _ = cache4(cache)
    dev = cache.get_device()
    if not isinstance(slots, torch.Tensor) or slots.dim() != 1:
        raise ValueError("slots must be a one-dimensional int32 tensor")
    t = slots.shape[0]
    at = vector(slots, "slots", torch.int32, t, dev)
    if k_out is None:
        k_out, ok = fresh(cache, t, n, dim, dtype)
    else:
        ok = heads(k_out, "k_out", dtype, dev, t, dim, n, True)
    if v_out is None:
        v_out, ov = fresh(cache, t, n, dim, dtype)
    else:
        ov = heads(v_out, "v_out", dtype, dev, t, dim, n, True)
    call(lib().vcclKv4Read, "vcclKv4Read", dev, c, at, ok, ov, t, DTYPES[dtype])
    return k_out, v_out


def kv4_attention(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor,
                  q_starts: torch.Tensor, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                  return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Causal attention of q [T, q heads, D] (bf16 or fp16) over the cache.

    Request b has rows q_starts[b] to q_starts[b + 1] of q and the kv_lens[b]
    tokens of the pages in block_table[b]; its last row sees all of them, the
    row before one less, and so on (the new tokens' keys and values are in the
    cache already).  q_starts must not fall.  q heads is a multiple of kv heads, head h reads key head
    h // (q heads / kv heads).  scale defaults to D ** -0.5.

    A row that sees nothing is 0 (lse -inf).  Rows behind the last request's
    are 0 (lse -inf) in a new output, and left as they are in ``out``.  Tokens
    on a page outside of the cache are not seen.  With return_lse also the
    natural logarithm of the sum of exponentials, f32 [T, q heads].
    """
    dev, dtype = float16s(q, "q"), q.dtype
    t, n, dim = q.shape
    c, kv_heads, _, page_size = cache4(cache, dim, dev)
    hq = heads(q, "q", dtype, dev, t, dim)
    if n % kv_heads:
        raise ValueError(f"{n} query heads do not divide over {kv_heads} key heads")
    if (not isinstance(block_table, torch.Tensor) or block_table.dtype != torch.int32 or block_table.dim() != 2
            or block_table.get_device() != dev or not block_table.is_contiguous() or 0 in block_table.shape):
        raise ValueError(f"block_table must be a contiguous int32 tensor [batch, pages per request] on CUDA device {dev}")
    batch, width = block_table.shape
    if batch > MAX_BATCH:
        raise ValueError(f"at most {MAX_BATCH} requests, got {batch}")
    if width * page_size > 2**30 or t * n > 2**31 - 1:
        raise ValueError("a request has at most 2^30 tokens, and the rows of all heads fit in 31 bits")
    a_kv = vector(kv_lens, "kv_lens", torch.int32, batch, dev)
    a_q = vector(q_starts, "q_starts", torch.int32, batch + 1, dev)
    new = out is None
    if new:
        out, ho = fresh(q, t, n, dim)
    else:
        ho = heads(out, "out", dtype, dev, t, dim, n, True)
    lse = q.new_empty((t, n), dtype=torch.float32) if return_lse else None
    h = lib()
    if current_device() == dev:
        size = h.vcclKv4AttentionWorkspace(batch, t, n, kv_heads, dim)
    else:  # the scratch goes by the device's SMs
        with on_device(dev):
            size = h.vcclKv4AttentionWorkspace(batch, t, n, kv_heads, dim)
    ws = cache.new_empty(size)
    call(h.vcclKv4Attention, "vcclKv4Attention", dev, hq, c, block_table.data_ptr(), width, a_kv, a_q, batch, t,
         dim ** -0.5 if scale is None else scale, ho, None if lse is None else lse.data_ptr(), 1 if new else 0,
         ws.data_ptr(), DTYPES[dtype])
    return (out, lse) if return_lse else out


def kv4_attention_status(device=None) -> None:
    """Raises VcclError if an attention launch on the device (default: the current one) gave up a wait, and forgets it.

    The kernels' waits are bounded; a launch that gave one up leaves its output
    incomplete.  The next ``kv4_attention`` raises this by itself.  A loop that
    replays a captured step makes no such call: synchronise, then ask here.
    """
    index = current_device() if device is None else torch.device(device).index
    with on_device(current_device() if index is None else index):
        result = lib().vcclKv4AttentionStatus()
    if result:
        _check(result, "vcclKv4Attention")
