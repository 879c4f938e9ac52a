# SPDX-License-Identifier: Apache-2.0
"""What the model operators (paging, rope, kv4) share: checks of tensors, and
the C structures of ``vccl_model.h`` as packed bytes.

A decode step makes several such calls per layer, so the host's time counts:
every attribute of a tensor is read once, devices are compared by number, and
a structure is packed in one step (half the time of a ctypes.Structure).
"""

from __future__ import annotations

import struct

import torch

from vkccl_b200.comm import DataType

DTYPES = {torch.bfloat16: int(DataType.BFLOAT16), torch.float16: int(DataType.FLOAT16),
          torch.float32: int(DataType.FLOAT32)}
_VECTOR = {torch.bfloat16: 8, torch.float16: 8, torch.float32: 4}  # elements in 16 bytes

_HEADS = struct.Struct("@Pqqi4x").pack       # vcclHeads_t: data, tokenStride, headStride, heads
_ROPE = struct.Struct("@PPPPiif4x").pack     # vcclRope_t: positions, invFreq, qWeight, kWeight, half, interleaved, eps
_KV4 = struct.Struct("@Piiii").pack          # vcclKv4_t: data, pages, pageSize, kvHeads, D


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# The same without the Stream object, where this torch has it.
stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)
current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


class on_device:
    """The library launches on the thread's current device: makes it ``index``."""

    __slots__ = ("_index", "_before")

    def __init__(self, index: int):
        self._index = index
        self._before = -1

    def __enter__(self):
        now = current_device()
        if now != self._index:
            self._before = now
            torch.cuda.set_device(self._index)

    def __exit__(self, *exc):
        if self._before >= 0:
            torch.cuda.set_device(self._before)


def call(fn, what: str, index: int, *args) -> None:
    """Calls a library entry on device ``index``, its current stream last."""
    if current_device() == index:
        result = fn(*args, stream(index))
    else:
        with on_device(index):
            result = fn(*args, stream(index))
    if result:
        from vkccl_b200.comm import _check

        _check(result, what)


def vector(t, name: str, dtype: torch.dtype, size: int, index: int) -> int:
    """A contiguous one-dimensional tensor of a fixed size on device ``index``; returns its address."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.shape != (size,) or t.get_device() != index:
        raise ValueError(f"{name} must be a {dtype} tensor of shape ({size},) on CUDA device {index}")
    if size > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def heads(t, name: str, dtype: torch.dtype, index: int, tokens: int, dim: int, n: int = 0,
          written: bool = False) -> bytes:
    """A [tokens, heads, D] tensor with contiguous channels and 16-byte vectors."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.get_device() != index or t.dim() != 3:
        raise ValueError(f"{name} must be a three-dimensional {dtype} tensor on CUDA device {index}")
    rows, count, width = t.shape
    if rows != tokens or width != dim or count < 1 or (n and count != n):
        raise ValueError(f"{name} has shape {tuple(t.shape)}; expected ({tokens}, {n or 'heads'}, {dim})")
    s0, s1, s2 = t.stride()
    if rows <= 1:
        s0 = 0
    if count <= 1:
        s1 = 0
    vec, at = _VECTOR[dtype], t.data_ptr()
    if s2 != 1 or s0 % vec or s1 % vec or at % 16 or s0 >= 2**31 or s1 >= 2**31 or count > 32768 or rows > 2**30:
        raise ValueError(f"{name} must have contiguous channels, token and head strides that are multiples of {vec} "
                         "elements below 2^31, a 16-byte aligned base, at most 32768 heads and 2^30 tokens")
    if written:
        (near, a), (far, b) = sorted(((s, c) for s, c in ((s0, rows), (s1, count))), key=lambda x: (x[1] > 1, x[0]))
        if (a > 1 and near < dim) or (b > 1 and far < (near * (a - 1) if a > 1 else 0) + dim):
            raise ValueError(f"{name} is written, and its rows overlap")
    return _HEADS(at, s0, s1, count)


def fresh(like: torch.Tensor, tokens: int, n: int, dim: int, dtype=None):
    """A new contiguous [tokens, n, D] tensor on like's device, in its type unless another is given, and its structure."""
    t = like.new_empty((tokens, n, dim), dtype=dtype)
    return t, _HEADS(t.data_ptr(), n * dim, dim, n)


def cache4(cache, dim: int = 0, index: int = -1):
    """A cache as ``kv4_alloc`` makes it (one layer's): (structure, kv heads, head dim, page size)."""
    if (not isinstance(cache, torch.Tensor) or cache.dtype != torch.uint8 or cache.dim() != 4 or not cache.is_cuda
            or not cache.is_contiguous()):
        raise ValueError("cache must be a contiguous uint8 CUDA tensor [pages, kv heads, page size / 16, 18 * head dim]")
    if index >= 0 and cache.get_device() != index:
        raise ValueError(f"cache must be on CUDA device {index}")
    pages, n, blocks, width = cache.shape
    at = cache.data_ptr()
    if (width != 18 * 64 and width != 18 * 128) or not (pages and n and blocks) or at % 16:
        raise ValueError(f"cache has shape {tuple(cache.shape)}; expected [pages, kv heads, page size / 16, 18 * head dim] "
                         "with a head dimension of 64 or 128, on a 16-byte aligned base")
    if dim and width != 18 * dim:
        raise ValueError(f"the cache holds heads of {width // 18} channels, the tensors of {dim}")
    if pages * blocks * 16 > 2**31 - 1:
        raise ValueError("a cache holds at most 2^31 - 1 slots")
    return _KV4(at, pages, blocks * 16, n, width // 18), n, width // 18, blocks * 16


def rope_of(positions, inv_freq, q_weight, k_weight, eps: float, interleaved: bool, dtype, index: int, tokens: int,
            dim: int) -> bytes:
    pos = vector(positions, "positions", torch.int32, tokens, index)
    if not isinstance(inv_freq, torch.Tensor) or inv_freq.dim() != 1:
        raise ValueError("inv_freq must be a one-dimensional tensor")
    half = inv_freq.shape[0]
    freq = vector(inv_freq, "inv_freq", torch.float32, half, index)
    if half < 8 or half % 8 or 2 * half > dim:
        raise ValueError(f"inv_freq has {half} frequencies; a multiple of 8 from 8 to head dim / 2 ({dim // 2}) is needed")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    wq = 0 if q_weight is None else vector(q_weight, "q_weight", dtype, dim, index)
    wk = 0 if k_weight is None else vector(k_weight, "k_weight", dtype, dim, index)
    if wq % 16 or wk % 16:
        raise ValueError("q_weight and k_weight must be 16-byte aligned")
    return _ROPE(pos, freq, wq, wk, half, 1 if interleaved else 0, eps)


def float16s(t, name: str) -> int:
    """A bf16 or fp16 [tokens, heads, D] tensor; returns its device's number."""
    if not isinstance(t, torch.Tensor) or (t.dtype != torch.bfloat16 and t.dtype != torch.float16) or not t.is_cuda or t.dim() != 3:
        raise ValueError(f"{name} must be a bf16 or fp16 CUDA tensor [tokens, heads, head dim]")
    return t.get_device()
