"""Attention over packed sequences of different lengths: grouped heads, causal
or not, forward and backward.

wan_flash_packed_fwd(q, k, v, q_offsets, k_offsets=None, causal=False) -> (o, lse)
wan_flash_packed_bwd(q, k, v, o, lse, do, q_offsets, k_offsets=None, causal=False) -> (dq, dk, dv)
wan_flash_attn_packed(q, k, v, q_offsets, k_offsets=None, causal=False) -> o   (autograd)

  q, o, do, dq  (total_q, h, 128) bf16: the sequences' rows one behind the other
  k, v, dk, dv  (total_k, h_kv, 128) bf16, h a multiple of h_kv: q head j reads
                key-value head j // (h // h_kv)
  lse           (h, total_q) fp32, natural log
  q_offsets     (n + 1) int32 on the device: sequence i is rows
                [q_offsets[i], q_offsets[i + 1]); k_offsets likewise for keys
                (default: the same)

Causal: query i of a sequence with lq queries and lk keys sees keys
j <= i + lk - lq (the last query sees every key).  A row that sees no key has
o = 0, lse = -inf and no gradient.  Rows outside every sequence (before the
first offset, behind the last) may hold anything: they reach no sequence's
result, and their o and gradients are 0, their lse -inf.

The offsets are read on the device only: nothing synchronises, and a captured
CUDA graph may be replayed with other offsets in the same tensors.  Offsets
that fall, or leave the tensor, give NaN everywhere, and
``wan_flash._lib.check_device()`` raises.  Contract violations that the host
can see raise AssertionError before any CUDA call.
"""

from __future__ import annotations

import ctypes

import torch

from wan_flash import _lib, features
from wan_flash.interface import _aligned, _ptr, _stream_ptr
from wan_flash.shapes import HEAD_DIM


def _check(q, k, v, q_offsets, k_offsets):
    k_offsets = q_offsets if k_offsets is None else k_offsets
    assert q.dtype == k.dtype == v.dtype == torch.bfloat16
    assert q.dim() == 3 and k.dim() == 3 and v.shape == k.shape
    assert q.shape[2] == HEAD_DIM and k.shape[2] == HEAD_DIM, "specialized for head_dim=128"
    h, h_kv = q.shape[1], k.shape[1]
    assert (h % h_kv == 0) if h_kv else h == 0, "q heads are a multiple of key-value heads"
    assert q_offsets.dtype == k_offsets.dtype == torch.int32
    assert q_offsets.dim() == 1 and q_offsets.shape == k_offsets.shape and q_offsets.numel() >= 1
    assert q.is_cuda and all(t.device == q.device for t in (k, v, q_offsets, k_offsets)), \
        "tensors must be on one CUDA device"
    return tuple(t if t.is_contiguous() else t.contiguous() for t in (q_offsets, k_offsets))


def _bytes(fn, *args) -> int:
    n = ctypes.c_size_t()
    _lib.check(fn(*args, ctypes.byref(n)))
    return n.value


def wan_flash_packed_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_offsets: torch.Tensor,
                         k_offsets: torch.Tensor | None = None, causal: bool = False):
    """(o, lse) of attention over packed sequences; see the module's text."""
    q_offsets, k_offsets = _check(q, k, v, q_offsets, k_offsets)
    q, k, v = (_aligned(t) for t in (q, k, v))
    total_q, h, _ = q.shape
    total_k, h_kv, _ = k.shape
    n = q_offsets.numel() - 1
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(h, total_q, device=q.device, dtype=torch.float32)
    if o.numel() == 0:
        return o, lse
    L = _lib.lib()
    size = _bytes(L.wf_packed_fwd_workspace, n, total_q)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device)
    with torch.cuda.device(q.device):
        rc = L.wf_packed_fwd(_ptr(q), _ptr(k), _ptr(v), _ptr(q_offsets), _ptr(k_offsets), _ptr(o), _ptr(lse), _ptr(ws),
                             size, n, total_q, total_k, h, h_kv, 1 if causal else 0,
                             ctypes.c_void_p(_stream_ptr(q.device)))
    _lib.check(rc)
    return o, lse


def wan_flash_packed_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
                         do: torch.Tensor, q_offsets: torch.Tensor, k_offsets: torch.Tensor | None = None,
                         causal: bool = False):
    """(dq, dk, dv) given the forward's o and lse and the gradient of o.

    dk and dv are bitwise reproducible; dq is accumulated with fp32 reductions
    unless ``features.set_bwd_overrides(deterministic=True)``.  ``nsplit`` of the
    backward features cuts the longest key tile's walk into that many pieces (0:
    the device chooses); the CTA-pair form does not apply."""
    q_offsets, k_offsets = _check(q, k, v, q_offsets, k_offsets)
    total_q, h, _ = q.shape
    total_k, h_kv, _ = k.shape
    assert o.dtype == do.dtype == torch.bfloat16 and o.shape == q.shape and do.shape == q.shape
    assert lse.dtype == torch.float32 and lse.shape == (h, total_q)
    assert all(t.device == q.device for t in (o, lse, do)), "tensors must be on one CUDA device"
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    if dq.numel() == 0 or dk.numel() == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    q, k, v, o, do = (_aligned(t) for t in (q, k, v, o, do))
    lse = lse if lse.is_contiguous() else lse.contiguous()
    n = q_offsets.numel() - 1
    f = features.get_bwd()
    cfg = _lib.PackedBwdCfg(min(int(f.nsplit), 1024), 1 if f.deterministic else 0)
    L = _lib.lib()
    with torch.cuda.device(q.device):
        size = _bytes(L.wf_packed_bwd_workspace, n, total_q, total_k, h, h_kv, ctypes.byref(cfg))
        ws = torch.empty(size, dtype=torch.uint8, device=q.device)
        rc = L.wf_packed_bwd(_ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), _ptr(do), _ptr(q_offsets), _ptr(k_offsets),
                             _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), size, n, total_q, total_k, h, h_kv,
                             1 if causal else 0, ctypes.byref(cfg), ctypes.c_void_p(_stream_ptr(q.device)))
    _lib.check(rc)
    return dq, dk, dv


class _WanFlashAttnPackedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_offsets, k_offsets, causal):
        o, lse = wan_flash_packed_fwd(q, k, v, q_offsets, k_offsets, causal)
        ctx.save_for_backward(q, k, v, o, lse, q_offsets, k_offsets)
        ctx.causal = causal
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, lse, q_offsets, k_offsets = ctx.saved_tensors
        dq, dk, dv = wan_flash_packed_bwd(q, k, v, o, lse, do, q_offsets, k_offsets, ctx.causal)
        return dq, dk, dv, None, None, None


def wan_flash_attn_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_offsets: torch.Tensor,
                          k_offsets: torch.Tensor | None = None, causal: bool = False):
    """Differentiable attention over packed sequences -> o (total_q, h, 128) bf16."""
    return _WanFlashAttnPackedFn.apply(q, k, v, q_offsets, q_offsets if k_offsets is None else k_offsets, bool(causal))
