# SPDX-License-Identifier: Apache-2.0
"""Llama-3-70B-shaped tensor-parallel decode step (hidden 8192, 80 layers).

Per layer and rank (TP = n, bf16, random-init weights):

    qkv   = x_norm @ W_qkv^T          [B, (64 + 2 * 8) * 128 / n]   column parallel
    attn  = qkv[:, :8192 / n]           (stand-in for attention over the KV cache)
    part  = attn @ W_o^T              [B, 8192]   row parallel -> partial sums
    x, x_norm = AllReduce(part) + x, RMSNorm(...)          <- fused kernel
    h     = silu(x_norm W_g^T) * (x_norm W_u^T)  [B, 28672 / n]  column parallel
    part  = h @ W_d^T                 [B, 8192]   row parallel -> partial sums
    x, x_norm = AllReduce(part) + x, RMSNorm(...)          <- fused kernel

so every layer does two all-reduces of [B, 8192] fused with the residual add
and RMSNorm (eps 1e-5), as in vLLM's TP decode.  ``step`` runs the 80
layers with this library's GEMMs and ``vcclAllReduceAddRMSNorm``;
``step_nccl`` runs the same layers with cuBLAS, NCCL all-reduce and a torch
RMSNorm.  The attention core of these two is replaced by a slice of the QKV
projection, identical in both paths, so the comparison isolates the TP
communication and the GEMMs.

``step_cached`` is the same step with its attention: each rank keeps its
kv_heads / n key heads in a paged cache held in 4 bits (``new_cache``), and a
step is one page plan, then per layer the projection, norm (with
``qk_norm``) and rotation of the new rows with their write to the cache in one
launch, and attention over the cache.  Prompts and single tokens go through it
alike, and it may be captured into a CUDA graph: lengths, pages and block
tables stay on the GPU.  ``return_plan`` tells which requests were refused.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Tuple, Union

import torch

from vkccl_b200.ops.fused import all_reduce_add_rms_norm
from vkccl_b200.ops.gemm import gemm_bf16, gemm_silu_mul, interleave_gate_up
from vkccl_b200.ops.kv4 import kv4_alloc, kv4_append_rope, kv4_attention
from vkccl_b200.ops.paging import PagePlan, plan_pages


@dataclass
class DecodeConfig:
    hidden: int = 8192
    intermediate: int = 28672
    heads: int = 64
    kv_heads: int = 8
    head_dim: int = 128
    layers: int = 80
    eps: float = 1e-5
    init_std: float = 0.02
    rope_theta: float = 500000.0
    qk_norm: bool = False  # norms of every query and key head before the rotation
    page_size: int = 64


@dataclass
class DecodeCache:
    """One rank's key/value cache: a 4-bit page pool per layer, which share the tables."""

    layers: List[torch.Tensor]  # uint8 [pages, kv heads of the rank, page size / 16, 18 * head dim]
    block_table: torch.Tensor   # int32 [requests, pages per request]
    lens: torch.Tensor          # int32 [requests] tokens cached
    free_pages: torch.Tensor    # int32 [pages] stack of free pages
    free_count: torch.Tensor    # int32 [1]
    page_size: int

    def plan(self, new_lens: torch.Tensor, rows: int, finished: Optional[torch.Tensor] = None) -> PagePlan:
        """Pages and slots for new_lens[i] more tokens of each request; the cache moves on."""
        return plan_pages(self.lens, new_lens, self.block_table, self.free_pages, self.free_count, self.page_size, rows,
                          finished=finished, lens_out=self.lens, count_out=self.free_count)


class TPLlamaDecode:
    def __init__(self, comm, cfg: DecodeConfig = DecodeConfig(), seed: int = 0, device: str = "cuda"):
        self.comm, self.cfg = comm, cfg
        n, r = comm.nranks, comm.rank
        h = cfg.hidden
        self.qkv_out = (cfg.heads + 2 * cfg.kv_heads) * cfg.head_dim // n
        self.attn_out = h // n
        self.inter = cfg.intermediate // n
        g = torch.Generator(device=device).manual_seed(seed * 7919 + r)

        def w(rows, cols):
            return (torch.randn(rows, cols, generator=g, device=device) * cfg.init_std).bfloat16()

        self.inv_freq = (cfg.rope_theta ** (-torch.arange(0, cfg.head_dim, 2, dtype=torch.float64) / cfg.head_dim)
                         ).float().to(device)
        self.layers = []
        for _ in range(cfg.layers):
            wg, wu = w(self.inter, h), w(self.inter, h)
            self.layers.append({
                "qkv": w(self.qkv_out, h),
                "o": w(h, self.attn_out),
                "gu": interleave_gate_up(wg, wu),
                "d": w(h, self.inter),
                "ln1": (1 + 0.02 * torch.randn(h, generator=g, device=device)).bfloat16(),
                "ln2": (1 + 0.02 * torch.randn(h, generator=g, device=device)).bfloat16(),
            })
            if cfg.qk_norm:
                for name in ("qn", "kn"):
                    self.layers[-1][name] = (1 + 0.02 * torch.randn(cfg.head_dim, generator=g, device=device)).bfloat16()

    def step(self, x: torch.Tensor, x_norm: torch.Tensor, n_layers: int | None = None) -> torch.Tensor:
        """One decode step; x (residual) is updated in place, returns the final normed state."""
        c = self.comm
        for L in self.layers[:n_layers]:
            qkv = gemm_bf16(x_norm, L["qkv"])
            part = gemm_bf16(qkv[:, : self.attn_out].contiguous(), L["o"])
            x_norm = all_reduce_add_rms_norm(c, part, x, L["ln1"], self.cfg.eps)
            hid = gemm_silu_mul(x_norm, L["gu"])
            part = gemm_bf16(hid, L["d"])
            x_norm = all_reduce_add_rms_norm(c, part, x, L["ln2"], self.cfg.eps)
        return x_norm

    def new_cache(self, requests: int, pages: int, max_tokens: int) -> DecodeCache:
        """A cache of `pages` pages for up to `requests` requests of at most max_tokens tokens."""
        c, dev = self.cfg, self.inv_freq.device
        if c.kv_heads % self.comm.nranks:
            raise ValueError(f"{c.kv_heads} key heads do not split over {self.comm.nranks} ranks")
        width = -(-max_tokens // c.page_size)
        return DecodeCache(
            [kv4_alloc(pages, c.page_size, c.kv_heads // self.comm.nranks, c.head_dim, device=dev) for _ in range(c.layers)],
            torch.full((requests, width), -1, dtype=torch.int32, device=dev),
            torch.zeros(requests, dtype=torch.int32, device=dev), torch.arange(pages, dtype=torch.int32, device=dev),
            torch.full((1,), pages, dtype=torch.int32, device=dev), c.page_size)

    def step_cached(self, x: torch.Tensor, x_norm: torch.Tensor, cache: DecodeCache, new_lens: torch.Tensor,
                    finished: Optional[torch.Tensor] = None, n_layers: int | None = None, return_plan: bool = False
                    ) -> Union[torch.Tensor, Tuple[torch.Tensor, PagePlan]]:
        """One step with attention over the cache.

        x, x_norm [rows, hidden] hold new_lens[i] (int32 [requests]) new rows of
        each request in order; rows behind them are padding.  finished
        (bool [requests]): requests that end, whose pages are free for this
        step.  x (residual) is updated in place; returns the final normed state.

        A request for which no pages are left, or whose rows or length do not
        fit, is refused: nothing of it is cached, and its rows come back
        without attention.  With return_plan also the step's plan, whose
        ``kv_lens`` is 0 where a request was refused (or holds nothing).
        """
        c, dim = self.cfg, self.cfg.head_dim
        n = self.comm.nranks
        hq, hk = c.heads // n, c.kv_heads // n
        plan = cache.plan(new_lens, x.shape[0], finished)
        for L, pages in zip(self.layers[:n_layers], cache.layers):
            qkv = gemm_bf16(x_norm, L["qkv"]).view(-1, hq + 2 * hk, dim)
            q = kv4_append_rope(pages, qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:], plan.slots, plan.positions,
                                self.inv_freq, q_weight=L.get("qn"), k_weight=L.get("kn"), eps=c.eps)
            attn = kv4_attention(q, pages, cache.block_table, plan.kv_lens, plan.q_starts)
            part = gemm_bf16(attn.view(-1, hq * dim), L["o"])
            x_norm = all_reduce_add_rms_norm(self.comm, part, x, L["ln1"], c.eps)
            hid = gemm_silu_mul(x_norm, L["gu"])
            part = gemm_bf16(hid, L["d"])
            x_norm = all_reduce_add_rms_norm(self.comm, part, x, L["ln2"], c.eps)
        return (x_norm, plan) if return_plan else x_norm

    def step_nccl(self, x: torch.Tensor, x_norm: torch.Tensor, group=None, n_layers: int | None = None) -> torch.Tensor:
        import torch.distributed as dist

        n = self.comm.nranks

        def ar_norm(part, weight):
            if n > 1:
                dist.all_reduce(part, group=group)
            x.add_(part)
            xf = x.float()
            return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + self.cfg.eps) * weight.float()).bfloat16()

        for L in self.layers[:n_layers]:
            qkv = x_norm @ L["qkv"].T
            part = qkv[:, : self.attn_out] @ L["o"].T
            x_norm = ar_norm(part, L["ln1"])
            gu = (x_norm @ L["gu"].T).view(-1, self.inter // 16, 2, 16)
            hid = (torch.nn.functional.silu(gu[:, :, 0]) * gu[:, :, 1]).reshape(-1, self.inter)
            part = hid @ L["d"].T
            x_norm = ar_norm(part, L["ln2"])
        return x_norm
