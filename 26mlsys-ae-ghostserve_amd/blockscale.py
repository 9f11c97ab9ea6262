"""A paged K/V cache in 8 or 4 bits with block scales.

No reference counterpart: the reference takes its cache from the engine that it
hooks, in 16 bits (bench_ghostserve_rdp.py:440-458).

  BlockPool   the pool: bytes that the codes, the copies to the host and the
              recovery take as they are
  read        tokens of it read back by slot, as K and V in 16 or 32 bits

:func:`.attention.norm_rotate_write` writes such a pool, :func:`.attention.prefix_attention`
attends over it, and :class:`.serving.PagedBackend` runs steps on it.

A token's K (or V) in a layer is a half record of bytes: kv_heads * dim codes
(8 bits: e4m3; 4 bits: e2m1, that is 0, .5, 1, 1.5, 2, 3, 4, 6 and a sign, two to a
byte, the first in the low half), then a scale byte for each block of 32
neighbouring values of a head, then up to 15 bytes that nothing writes, to a multiple
of 16.  A value is code * 2^(byte - 127); byte 255 makes all 32 NaN.  That is 8.25 or
4.25 bits a value.  A block's scale is the smallest power of two with which no value
passes the largest code (448 or 6); codes are the nearest ones, ties to even.  Values
that would round past the largest of the type they come from are taken as the last that
does not: for float16 those past 61440 (8 bits) or 49152 (4 bits, down by up to a
quarter), for bfloat16 and float32 past 1.875 or 1.5 times 2^127.  No others are clipped.
A block in which a value is infinite or NaN reads back as NaN.
"""
from __future__ import annotations

import torch

from . import _lib

_BLOCK = 32
_CODES = {8: 4, 4: 5}                  # bits -> KVEC_BLOCK_* of include/kvec.h
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def half_bytes(kv_heads: int, dim: int, bits: int) -> int:
    """Bytes of K (or V) of one token in one layer."""
    if bits not in _CODES:
        raise ValueError("bits must be 8 or 4")
    if kv_heads < 1 or dim < _BLOCK or dim % _BLOCK or dim > 256:
        raise ValueError("kv_heads must be positive, dim a multiple of 32 up to 256")
    n = kv_heads * dim
    return (n * bits // 8 + n // _BLOCK + 15) // 16 * 16


class BlockPool:
    """A paged K/V pool in ``bits`` (8 or 4) with block scales, over ``data``: uint8
    [layers, pool_pages, page_tokens, 2 (K,V), half_bytes(kv_heads, dim, bits)], contiguous.

    ``shape`` is that of a pool of plain values: (layers, pool_pages, page_tokens, 2,
    kv_heads, dim).  ``records`` is the pool as :class:`.paged.PagedKV` codes it."""

    __slots__ = ("data", "bits", "kv_heads", "dim", "shape")

    def __init__(self, data: torch.Tensor, kv_heads: int, dim: int, bits: int = 8):
        size = data.shape
        half = half_bytes(kv_heads, dim, bits)
        if len(size) != 5 or size[3] != 2 or size[4] != half or data.dtype != torch.uint8:
            raise ValueError(f"data must be uint8 [layers, pool_pages, page_tokens, 2, {half}]")
        if not data.is_contiguous():
            raise ValueError("data must be contiguous")
        self.data, self.bits, self.kv_heads, self.dim = data, bits, kv_heads, dim
        self.shape = (size[0], size[1], size[2], 2, kv_heads, dim)

    @classmethod
    def zeros(cls, layers: int, pool_pages: int, page_tokens: int, kv_heads: int, dim: int, bits: int = 8,
              device="cuda") -> "BlockPool":
        """An empty pool (every value 0)."""
        size = (layers, pool_pages, page_tokens, 2, half_bytes(kv_heads, dim, bits))
        return cls(torch.zeros(size, dtype=torch.uint8, device=device), kv_heads, dim, bits)

    @property
    def records(self) -> torch.Tensor:
        """The pool's bytes, [layers, pool_pages, page_tokens, 2, 1, half_bytes]."""
        return self.data.unsqueeze(4)

    @property
    def device(self) -> torch.device:
        return self.data.device

    def layer(self, layer: int) -> tuple[int, int]:
        """(address, slots) of a layer."""
        L, pages, pt, _, _, _ = self.shape
        if not 0 <= layer < L:
            raise ValueError(f"layer {layer} not in [0, {L})")
        return self.data.data_ptr() + layer * self.data.stride(0), pages * pt

    @property
    def code(self) -> int:
        """KVEC_BLOCK_* of include/kvec.h."""
        return _CODES[self.bits]


def read(pool: BlockPool, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16, *, layer: int = 0,
         out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V, [tokens, kv_heads, dim] each, of the tokens at ``slots`` (int32, page *
    page_tokens + place) of the pool's ``layer``, in float32, bfloat16 or float16.

    A token whose slot is negative or past the pool is zeros.  bfloat16 holds every value
    of such a pool but those under 2^-126; float16 makes values past 65504 infinite.
    ``out``: an earlier result, or two contiguous tensors like it, written again.  Nothing
    is read back to the host, so the call can be captured in a graph."""
    if not isinstance(pool, BlockPool):
        raise ValueError("read takes a BlockPool")
    if slots.dim() != 1 or slots.dtype != torch.int32 or not slots.is_contiguous():
        raise ValueError("slots must be contiguous int32 [tokens]")
    if dtype not in _TYPES:
        raise ValueError("dtype must be float32, bfloat16 or float16")
    dev, N = slots.device, slots.shape[0]
    base, n_slots = pool.layer(layer)
    size = (N, pool.kv_heads, pool.dim)
    if out is None:
        _lib.require_same_device(dev, pool.data, what="read tensor")
        k, v = slots.new_empty((2, *size), dtype=dtype).unbind(0)
    else:
        k, v = out
        _lib.require_same_device(dev, pool.data, k, v, what="read tensor")
        _lib.require_no_grad(k, v, what="read")
        for t in out:
            if t.shape != size or t.dtype != dtype or not t.is_contiguous():
                raise ValueError(f"out must be two contiguous tensors of {size} and dtype")
    s = _lib.pack(_lib.BLOCK_READ_FORMAT, N, pool.kv_heads, pool.dim, pool.code, base, n_slots, slots.data_ptr(),
                  _TYPES[dtype], k.data_ptr(), v.data_ptr())
    _lib.call_on(dev, "kvec_block_read_kv", s, _lib.stream_handle(dev))
    return k, v
