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

Contract violations raise AssertionError before any CUDA call.  The caches
are read by their strides and never copied.  Lengths and page numbers are
device data: an impossible one gives NaN in its sequence's outputs, and
``wan_flash._lib.check_device()`` raises.  Lengths and pages may change
between replays of a captured CUDA graph; shapes may not.
"""

from __future__ import annotations

import ctypes

import torch

from wan_flash import _lib
from wan_flash.interface import _aligned, _ptr, _stream_ptr
from wan_flash.shapes import HEAD_DIM

_WORKSPACE_BYTES: dict = {}  # (device index, h, h_kv) -> bytes


def _workspace_bytes(device: torch.device, h: int, h_kv: int) -> int:
    key = (device.index, h, h_kv)
    if key not in _WORKSPACE_BYTES:
        n = ctypes.c_size_t()
        _lib.check(_lib.lib().wf_decode_workspace(h, h_kv, ctypes.byref(n)))
        _WORKSPACE_BYTES[key] = n.value
    return _WORKSPACE_BYTES[key]


def wan_flash_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                     lengths: torch.Tensor):
    """One new token per sequence over the paged cache -> (o, lse); see the module's text.

    A sequence of length 0 gives o = 0 and lse = -inf.  k_cache and v_cache may be
    strided views (of one tensor that holds both, say) as long as rows of 128
    are contiguous and 16-byte aligned."""
    assert q.dtype == k_cache.dtype == v_cache.dtype == torch.bfloat16
    assert q.dim() == 3 and k_cache.dim() == 4 and k_cache.shape == v_cache.shape
    b, h, d = q.shape
    n_pages, page_size, h_kv, dk = k_cache.shape
    assert d == HEAD_DIM and dk == HEAD_DIM, "specialized for head_dim=128"
    assert h_kv > 0 and h % h_kv == 0, "q heads are a multiple of key-value heads"
    assert page_size > 0
    assert page_table.dtype == torch.int32 and page_table.dim() == 2 and page_table.shape[0] == b
    assert lengths.dtype == torch.int32 and lengths.shape == (b,)
    assert page_table.shape[1] * page_size <= 2**31 - 1025
    for x in (k_cache, v_cache):
        assert x.stride(-1) == 1 and x.data_ptr() % 16 == 0 and all(s % 8 == 0 and s >= 0 for s in x.stride()[:-1]), \
            "cache rows of 128 must be contiguous and 16-byte aligned"
    assert q.is_cuda and all(t.device == q.device for t in (k_cache, v_cache, page_table, lengths)), \
        "tensors must be on one CUDA device"
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(b, h, device=q.device, dtype=torch.float32)
    if o.numel() == 0:
        return o, lse
    q = _aligned(q)
    lengths = lengths if lengths.is_contiguous() else lengths.contiguous()
    page_table = page_table if page_table.stride(1) == 1 or page_table.shape[1] <= 1 else page_table.contiguous()
    cfg = _lib.DecodeCfg(n_pages, page_size, page_table.shape[1], 0, page_table.stride(0), *k_cache.stride()[:3],
                         *v_cache.stride()[:3])
    with torch.cuda.device(q.device):
        n = _workspace_bytes(q.device, h, h_kv)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        rc = _lib.lib().wf_decode(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(page_table), _ptr(lengths), _ptr(o),
                                  _ptr(lse), _ptr(ws), n, b, h, h_kv, ctypes.byref(cfg),
                                  ctypes.c_void_p(_stream_ptr(q.device)))
    _lib.check(rc)
    return o, lse
