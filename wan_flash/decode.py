"""Attention of one new token per sequence over a paged key-value cache.

wan_flash_decode(q, k_cache, v_cache, page_table, lengths) -> (o, lse)
  q (b, h, 128) bf16: the new token's queries
  k_cache, v_cache (n_pages, page_size, h_kv, 128) bf16
  page_table (b, max_pages) int32, lengths (b) int32
  o (b, h, 128) bf16, lse (b, h) fp32 natural log

The serving form of causal attention (``wan_flash.packed``): the new token's
key and value are written to the cache first (``lengths`` counts them), then
its queries see everything cached.  Token t of sequence i is slot
t % page_size of page page_table[i, t // page_size]; writing it is a plain
index assignment, ``k_cache[page, slot] = k``.

Contract violations raise AssertionError before any CUDA call.  There is no
backward: serving only, and o never asks for a gradient, nor has it a
forward-mode tangent.  The caches are read
by their strides and never copied.  Lengths and page numbers are
device data: an impossible one gives NaN in its sequence's outputs, and
``wan_flash._lib.check_device()`` raises.  Lengths and pages may change
between replays of a captured CUDA graph; shapes may not.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from wan_flash import _lib
from wan_flash.interface import _aligned, _launch
from wan_flash.shapes import HEAD_DIM


@functools.lru_cache(maxsize=256)
def _workspace_bytes(index: int, b: int, h: int, h_kv: int, max_pages: int, page_size: int) -> int:
    """Of device `index`."""
    size = ctypes.c_size_t()
    with torch.cuda.device(index):
        _lib.check(_lib.lib().wf_decode_workspace(b, h, h_kv, max_pages, page_size, ctypes.byref(size)))
    return size.value


@functools.lru_cache(maxsize=256)
def _cfg(*sizes):
    """The C options of a cache's shape and strides (1.2 us to make, 0.2 to find)."""
    return _lib.DecodeCfg(*sizes)


def wan_flash_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                     lengths: torch.Tensor):
    """One new token per sequence over the paged cache -> (o, lse); see the module's text.

    A sequence of length 0 gives o = 0 and lse = -inf.  k_cache and v_cache may be
    strided views (of one tensor that holds both, say) as long as rows of 128
    are contiguous and 16-byte aligned."""
    assert q.dtype is torch.bfloat16 and k_cache.dtype is torch.bfloat16 and v_cache.dtype is torch.bfloat16
    assert q.dim() == 3 and k_cache.dim() == 4 and k_cache.shape == v_cache.shape
    b, h, d = q.shape
    n_pages, page_size, h_kv, dk = k_cache.shape
    assert d == HEAD_DIM and dk == HEAD_DIM, "specialized for head_dim=128"
    assert h_kv > 0 and h % h_kv == 0, "q heads are a multiple of key-value heads"
    assert page_size > 0
    assert page_table.dtype is torch.int32 and page_table.dim() == 2 and page_table.shape[0] == b
    assert lengths.dtype is torch.int32 and lengths.shape == (b,)
    width = page_table.shape[1]
    assert width * page_size <= 2**31 - 1025
    ks, vs = k_cache.stride(), v_cache.stride()
    k_ptr, v_ptr = k_cache.data_ptr(), v_cache.data_ptr()
    assert ks[3] == 1 and vs[3] == 1 and (k_ptr | v_ptr) % 16 == 0 and \
        (ks[0] | ks[1] | ks[2] | vs[0] | vs[1] | vs[2]) % 8 == 0, "cache rows of 128 must be contiguous and 16-byte aligned"
    device = q.device
    assert q.is_cuda and k_cache.device == device and v_cache.device == device and page_table.device == device and \
        lengths.device == device, "tensors must be on one CUDA device"
    q = _aligned(q)
    o = torch.empty_like(q)
    lse = q.new_empty((b, h), dtype=torch.float32)
    if b == 0 or h == 0:
        return o, lse
    lengths = lengths.contiguous()
    if width > 1 and page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    cfg = _cfg(n_pages, page_size, width, 0, page_table.stride(0), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2])
    size = _workspace_bytes(device.index, b, h, h_kv, width, page_size)
    ws = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _launch(_lib.lib().wf_decode, device, q.data_ptr(), k_ptr, v_ptr, page_table.data_ptr(), lengths.data_ptr(),
            o.data_ptr(), lse.data_ptr(), ws.data_ptr() if size else None, size, b, h, h_kv, cfg)
    return o, lse
