# SPDX-License-Identifier: Apache-2.0
"""What the model operators (paging, rope, kv4) share: checks of tensors, and
the C structures of ``vccl_model.h``."""

from __future__ import annotations

import ctypes

import torch

from vkccl_b200.comm import DataType

DTYPES = {torch.bfloat16: int(DataType.BFLOAT16), torch.float16: int(DataType.FLOAT16),
          torch.float32: int(DataType.FLOAT32)}


class Heads(ctypes.Structure):
    """``vcclHeads_t``: a [tokens, heads, D] tensor."""

    _fields_ = [("data", ctypes.c_void_p), ("tokenStride", ctypes.c_longlong), ("headStride", ctypes.c_longlong),
                ("heads", ctypes.c_int)]


class Rope(ctypes.Structure):
    """``vcclRope_t``."""

    _fields_ = [("positions", ctypes.c_void_p), ("invFreq", ctypes.c_void_p), ("qWeight", ctypes.c_void_p),
                ("kWeight", ctypes.c_void_p), ("half", ctypes.c_int), ("interleaved", ctypes.c_int),
                ("eps", ctypes.c_float)]


class Kv4(ctypes.Structure):
    """``vcclKv4_t``: the 4-bit cache of one layer."""

    _fields_ = [("data", ctypes.c_void_p), ("pages", ctypes.c_int), ("pageSize", ctypes.c_int),
                ("kvHeads", ctypes.c_int), ("D", ctypes.c_int)]


class on_device:
    """The library launches on the thread's current device: makes it ``dev``'s."""

    __slots__ = ("_index", "_before")

    def __init__(self, dev: torch.device):
        self._index = dev.index
        self._before = -1

    def __enter__(self):
        now = torch.cuda.current_device()
        if now != self._index:
            self._before = now
            torch.cuda.set_device(self._index)

    def __exit__(self, *exc):
        if self._before >= 0:
            torch.cuda.set_device(self._before)


def stream(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def vector(t, name: str, dtype: torch.dtype, size: int, dev: torch.device) -> int:
    """A contiguous one-dimensional tensor of a fixed size; returns its address."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != 1 or t.shape[0] != size or t.device != dev:
        raise ValueError(f"{name} must be a {dtype} tensor of shape ({size},) on {dev}")
    if size > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def heads(t, name: str, dtype: torch.dtype, dev: torch.device, tokens: int, dim: int, n: int = 0,
          written: bool = False) -> Heads:
    """A [tokens, heads, D] tensor with contiguous channels and 16-byte vectors."""
    if not isinstance(t, torch.Tensor) or t.dim() != 3 or t.dtype != dtype or t.device != dev:
        raise ValueError(f"{name} must be a three-dimensional {dtype} tensor on {dev}")
    rows, count, width = t.shape
    if rows != tokens or width != dim or count < 1 or (n and count != n):
        raise ValueError(f"{name} has shape {tuple(t.shape)}; expected ({tokens}, {n or 'heads'}, {dim})")
    s0, s1, s2 = t.stride()
    s0, s1 = (s0 if rows > 1 else 0), (s1 if count > 1 else 0)
    vec = 16 // t.element_size()
    if s2 != 1 or s0 % vec or s1 % vec or (rows and t.data_ptr() % 16):
        raise ValueError(f"{name} must have contiguous channels, token and head strides that are multiples of {vec} "
                         "elements and a 16-byte aligned base")
    if written:
        a, b = (s0, rows), (s1, count)
        small, large = (a, b) if b[1] <= 1 or (a[1] > 1 and a[0] <= b[0]) else (b, a)
        if (small[1] > 1 and small[0] < dim) or (large[1] > 1 and small[1] > 1 and large[0] < small[0] * (small[1] - 1) + dim):
            raise ValueError(f"{name} is written, and its rows overlap")
    return Heads(t.data_ptr(), s0, s1, count)


def cache4(cache, dim: int = 0, dev=None) -> Kv4:
    """A cache as ``kv4_alloc`` makes it (one layer's)."""
    if (not isinstance(cache, torch.Tensor) or cache.dtype != torch.uint8 or cache.dim() != 4 or not cache.is_cuda
            or not cache.is_contiguous() or cache.data_ptr() % 16):
        raise ValueError("cache must be a contiguous uint8 CUDA tensor [pages, kv heads, page size / 16, 18 * head dim]")
    if dev is not None and cache.device != dev:
        raise ValueError(f"cache must be on {dev}")
    pages, n, blocks, width = cache.shape
    if width not in (18 * 64, 18 * 128) or not (pages and n and blocks):
        raise ValueError(f"cache has shape {tuple(cache.shape)}; expected [pages, kv heads, page size / 16, 18 * head dim] "
                         "with a head dimension of 64 or 128")
    if dim and width != 18 * dim:
        raise ValueError(f"the cache holds heads of {width // 18} channels, the tensors of {dim}")
    if pages * blocks * 16 > 2**31 - 1:
        raise ValueError("a cache holds at most 2^31 - 1 slots")
    return Kv4(cache.data_ptr(), pages, blocks * 16, n, width // 18)


def rope_of(positions, inv_freq, q_weight, k_weight, eps: float, interleaved: bool, dtype, dev, tokens: int,
            dim: int) -> Rope:
    pos = vector(positions, "positions", torch.int32, tokens, dev)
    if not isinstance(inv_freq, torch.Tensor) or inv_freq.dim() != 1:
        raise ValueError("inv_freq must be a one-dimensional tensor")
    half = inv_freq.shape[0]
    freq = vector(inv_freq, "inv_freq", torch.float32, half, dev)
    if half < 8 or half % 8 or 2 * half > dim:
        raise ValueError(f"inv_freq has {half} frequencies; a multiple of 8 from 8 to head dim / 2 ({dim // 2}) is needed")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    weights = []
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        weights.append(None if w is None else vector(w, name, dtype, dim, dev))
        if w is not None and weights[-1] % 16:
            raise ValueError(f"{name} must be 16-byte aligned")
    return Rope(pos, freq, weights[0], weights[1], half, int(bool(interleaved)), float(eps))


def float16s(t, name: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in (torch.bfloat16, torch.float16) or t.dim() != 3:
        raise ValueError(f"{name} must be a bf16 or fp16 CUDA tensor [tokens, heads, head dim]")
