# SPDX-License-Identifier: Apache-2.0
"""Block tables and slots of a serving step, built on the GPU.

plan_pages(lens, new_lens, block_table, free_pages, free_count, page_size, tokens, finished=None)
    One call at the start of a step (stream-ordered, no host synchronisation,
    fit for a CUDA graph): finished requests give their pages back, requests
    with new tokens take the pages they need, and every row of the batch gets
    its position, slot and request.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from vkccl_b200._lib import lib
from vkccl_b200.ops._args import call, vector

MAX_BATCH = 8192


@dataclass
class PagePlan:
    """One step's rows.  A request is granted if its pages were there; a refused one keeps its length and has no rows to
    attend with (``kv_lens`` 0, slots -1)."""

    positions: torch.Tensor   # [tokens] int32 position of the row in its request
    slots: torch.Tensor       # [tokens] int32 page * page_size + place; -1 for refused requests and padding
    requests: torch.Tensor    # [tokens] int32; -1 for rows behind the last request's
    q_starts: torch.Tensor    # [batch + 1] int32 first row of each request
    kv_lens: torch.Tensor     # [batch] int32 tokens to attend to, the new ones included; 0 where refused
    lens: torch.Tensor        # [batch] int32 tokens cached after this step
    free_count: torch.Tensor  # [1] int32 pages left on the stack


def plan_pages(lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
               free_count: torch.Tensor, page_size: int, tokens: int, finished: Optional[torch.Tensor] = None,
               lens_out: Optional[torch.Tensor] = None, count_out: Optional[torch.Tensor] = None) -> PagePlan:
    """Rows, slots and pages of one step.

    lens [batch] (int32) tokens cached per request, new_lens [batch] tokens
    that each brings now, finished [batch] (bool or uint8) those that end:
    their pages go back first, and their length counts as 0.  block_table
    [batch, width] and the stack free_pages[:free_count] are updated in place;
    request i takes ceil((L + n) / page_size) - ceil(L / page_size) pages.  A
    request is refused if its length would not fit the table, its rows would
    not fit in ``tokens`` (the padded number of rows), or the pages that the
    requests up to it ask for are not there.  ``lens`` and ``free_count`` are
    left as they are unless passed again as ``lens_out`` and ``count_out``.
    """
    if not isinstance(lens, torch.Tensor) or not lens.is_cuda or lens.dim() != 1:
        raise ValueError("lens must be a one-dimensional int32 CUDA tensor")
    dev, batch = lens.get_device(), lens.shape[0]
    if not 1 <= batch <= MAX_BATCH:
        raise ValueError(f"1 to {MAX_BATCH} requests, got {batch}")
    if (not isinstance(block_table, torch.Tensor) or block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != batch
            or block_table.shape[1] < 1 or block_table.get_device() != dev or not block_table.is_contiguous()):
        raise ValueError(f"block_table must be a contiguous int32 tensor [{batch}, pages per request] on CUDA device {dev}")
    width = block_table.shape[1]
    if not isinstance(free_pages, torch.Tensor) or free_pages.dim() != 1 or free_pages.shape[0] < 1:
        raise ValueError("free_pages must be a one-dimensional int32 tensor with room for every page")
    pool, page_size, tokens = free_pages.shape[0], int(page_size), int(tokens)
    if page_size < 1 or not 0 <= tokens <= 2**30 or pool * page_size > 2**31 - 1 or width * page_size > 2**31 - 1:
        raise ValueError("page_size must be positive, tokens 0 to 2^30, and slots and lengths fit in 31 bits")
    i32 = torch.int32
    a_lens, a_new = vector(lens, "lens", i32, batch, dev), vector(new_lens, "new_lens", i32, batch, dev)
    a_free, a_count = vector(free_pages, "free_pages", i32, pool, dev), vector(free_count, "free_count", i32, 1, dev)
    a_done = None
    if finished is not None:
        if not isinstance(finished, torch.Tensor) or finished.dtype not in (torch.bool, torch.uint8):
            raise ValueError("finished must be bool or uint8")
        a_done = vector(finished, "finished", finished.dtype, batch, dev)
    buffer = lens.new_empty(3 * tokens + 5 * batch + 3)
    base = buffer.data_ptr()
    positions, slots, requests, q_starts, kv_lens, after, count, _ = buffer.split(
        (tokens, tokens, tokens, batch + 1, batch, batch, 1, 2 * batch + 1))
    at = base + 12 * tokens
    a_after, a_left = at + 4 * (2 * batch + 1), at + 4 * (3 * batch + 1)
    if lens_out is not None:
        after, a_after = lens_out, vector(lens_out, "lens_out", i32, batch, dev)
    if count_out is not None:
        count, a_left = count_out, vector(count_out, "count_out", i32, 1, dev)
    call(lib().vcclPagePlan, "vcclPagePlan", dev, a_lens, a_new, a_done, block_table.data_ptr(), a_free, a_count, batch,
         width, pool, page_size, tokens, base, base + 4 * tokens, base + 8 * tokens, at, at + 4 * (batch + 1), a_after,
         a_left, at + 4 * (3 * batch + 2))
    return PagePlan(positions, slots, requests, q_starts, kv_lens, after, count)
