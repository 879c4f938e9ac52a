# SPDX-License-Identifier: Apache-2.0
"""RMS norm of query and key heads and the position rotation, in one pass.

qk_norm_rope(q, k, positions, inv_freq, q_weight=None, k_weight=None)
    x / sqrt(mean(x^2) + eps) * weight for every head where a weight is given,
    then the first 2 * len(inv_freq) channels rotate by position * inv_freq.
qk_norm_rope_backward(dq, dk, q, k, positions, inv_freq, ...)
    its gradients, with those of the weights.

Tensors are [tokens, heads, head dim] in bf16 or fp16, with any token and head
strides that are multiples of 8 elements: slices of one projection's output
need no copy.  The angle is taken in 64 bits, so far positions keep it.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from vkccl_b200._lib import lib
from vkccl_b200.ops._args import DTYPES, call, float16s, fresh, heads, rope_of


def _sizes(q: torch.Tensor, k: torch.Tensor):
    dev = float16s(q, "q")
    t, n, dim = q.shape
    if dim % 8 or not 16 <= dim <= 256:
        raise ValueError(f"the head dimension must be a multiple of 8 from 16 to 256, got {dim}")
    if not isinstance(k, torch.Tensor) or k.dim() != 3:
        raise ValueError("k must be a tensor [tokens, heads, head dim]")
    return dev, q.dtype, t, n, k.shape[1], dim


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Norm and rotation of q [T, q heads, D] and k [T, k heads, D].

    positions [T] int32, inv_freq f32 [rotated / 2] (a multiple of 8), weights
    [D] in q's type or None (no norm).  interleaved: channels (2j, 2j + 1) turn
    together, else (j, j + rotated / 2).  An output may be its input; it must
    not overlap it in another way.

    There is no autograd history: in grad mode q, k and weights that require a
    gradient are refused.  Train with the call in torch.no_grad() (or in an
    autograd.Function's forward) and ``qk_norm_rope_backward``.
    """
    if torch.is_grad_enabled():
        for x in (q, k, q_weight, k_weight):
            if getattr(x, "requires_grad", False):
                raise ValueError("qk_norm_rope has no autograd history, and an input requires a gradient: call it in "
                                 "torch.no_grad(), and qk_norm_rope_backward for the gradients")
    dev, dtype, t, nq, nk, dim = _sizes(q, k)
    hq, hk = heads(q, "q", dtype, dev, t, dim), heads(k, "k", dtype, dev, t, dim)
    rope = rope_of(positions, inv_freq, q_weight, k_weight, eps, interleaved, dtype, dev, t, dim)
    if q_out is None:
        q_out, oq = fresh(q, t, nq, dim)
    else:
        oq = heads(q_out, "q_out", dtype, dev, t, dim, nq, True)
    if k_out is None:
        k_out, ok = fresh(k, t, nk, dim)
    else:
        ok = heads(k_out, "k_out", dtype, dev, t, dim, nk, True)
    call(lib().vcclQkNormRope, "vcclQkNormRope", dev, hq, hk, rope, oq, ok, t, dim, DTYPES[dtype])
    return q_out, k_out


def qk_norm_rope_backward(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
                          inv_freq: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                          k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                          dq_in: Optional[torch.Tensor] = None, dk_in: Optional[torch.Tensor] = None
                          ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Gradients of ``qk_norm_rope`` from dq, dk (of its outputs) and q, k (its inputs).

    Returns (dq_in, dk_in, dq_weight, dk_weight); a weight's gradient is None
    where there is no weight.  The sums over tokens and heads are f32 (their
    join f64) in a fixed order: the same bits on every run.  dq_in may be dq,
    dk_in may be dk.
    """
    dev, dtype, t, nq, nk, dim = _sizes(q, k)
    hq, hk = heads(q, "q", dtype, dev, t, dim), heads(k, "k", dtype, dev, t, dim)
    gq, gk = heads(dq, "dq", dtype, dev, t, dim, nq), heads(dk, "dk", dtype, dev, t, dim, nk)
    rope = rope_of(positions, inv_freq, q_weight, k_weight, eps, interleaved, dtype, dev, t, dim)
    if dq_in is None:
        dq_in, oq = fresh(q, t, nq, dim)
    else:
        oq = heads(dq_in, "dq_in", dtype, dev, t, dim, nq, True)
    if dk_in is None:
        dk_in, ok = fresh(k, t, nk, dim)
    else:
        ok = heads(dk_in, "dk_in", dtype, dev, t, dim, nk, True)
    dwq = None if q_weight is None else q_weight.new_empty(dim)
    dwk = None if k_weight is None else k_weight.new_empty(dim)
    h, ws = lib(), None
    if dwq is not None or dwk is not None:
        ws = torch.empty(h.vcclQkNormRopeBackwardWorkspace(dim), dtype=torch.uint8, device=q.device)
    call(h.vcclQkNormRopeBackward, "vcclQkNormRopeBackward", dev, gq, gk, hq, hk, rope, oq, ok,
         None if dwq is None else dwq.data_ptr(), None if dwk is None else dwk.data_ptr(),
         None if ws is None else ws.data_ptr(), t, dim, DTYPES[dtype])
    return dq_in, dk_in, dwq, dwk
