"""Attention over packed sequences of different lengths: grouped heads, causal
or not, forward and backward.

wan_flash_packed_fwd(q, k, v, q_offsets, k_offsets=None, causal=False) -> (o, lse[, o_residual])
wan_flash_packed_bwd(q, k, v, o, lse, do, q_offsets, k_offsets=None, causal=False, o_residual=None) -> (dq, dk, dv)
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
CUDA graph may be replayed with other offsets in the same tensors.  (A training
step is captured while no autograd graph from outside the capture holds the
same leaves: their gradient accumulation would wait on that graph's stream.)
Offsets that fall, or leave the tensor, give NaN everywhere, and
``wan_flash._lib.check_device()`` raises.  Contract violations that the host
can see raise AssertionError before any CUDA call.
"""

from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable

from wan_flash import _lib, features
from wan_flash.interface import _aligned, _has_tangent, _launch
from wan_flash.shapes import HEAD_DIM


def _check(q, k, v, q_offsets, k_offsets):
    assert q.dtype is torch.bfloat16 and k.dtype is torch.bfloat16 and v.dtype is torch.bfloat16
    assert q.dim() == 3 and k.dim() == 3 and v.shape == k.shape
    total_q, h, d = q.shape
    total_k, h_kv, dk = k.shape
    assert d == HEAD_DIM and dk == HEAD_DIM, "specialized for head_dim=128"
    assert (h % h_kv == 0) if h_kv else h == 0, "q heads are a multiple of key-value heads"
    assert q_offsets.dtype is torch.int32 and k_offsets.dtype is torch.int32
    assert q_offsets.dim() == 1 and q_offsets.shape == k_offsets.shape and q_offsets.numel() >= 1
    device = q.device
    assert q.is_cuda and k.device == device and v.device == device and q_offsets.device == device and \
        k_offsets.device == device, "tensors must be on one CUDA device"
    return total_q, total_k, h, h_kv, q_offsets.numel() - 1, device


@functools.lru_cache(maxsize=256)
def _fwd_bytes(index: int, n: int, total_q: int, total_k: int, h: int) -> int:
    """The workspace's size on device `index`."""
    size = ctypes.c_size_t()
    with torch.cuda.device(index):
        _lib.check(_lib.lib().wf_packed_fwd_workspace(n, total_q, total_k, h, ctypes.byref(size)))
    return size.value


@functools.lru_cache(maxsize=16)
def _fwd_cfg(rescale_skip_threshold: float, num_sms: int):
    """The C options of the forward's features that apply."""
    return _lib.FwdCfg(rescale_skip_threshold, 0, num_sms, 0)


@functools.lru_cache(maxsize=256)
def _bwd_cfg_bytes(index: int, n: int, total_q: int, total_k: int, h: int, h_kv: int, nsplit: int, deterministic: bool,
                   pdl: bool):
    """The C options and the workspace's size on device `index`."""
    sizes, size = _lib.PackedBwdCfg(min(nsplit, 1024), 1 if deterministic else 0), ctypes.c_size_t()
    with torch.cuda.device(index):
        _lib.check(_lib.lib().wf_packed_bwd_workspace(n, total_q, total_k, h, h_kv, ctypes.byref(sizes),
                                                      ctypes.byref(size)))
    return _lib.BwdCfg(sizes.nsplit, 1, sizes.deterministic, 0 if pdl else 1), size.value


def wan_flash_packed_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_offsets: torch.Tensor,
                         k_offsets: torch.Tensor | None = None, causal: bool = False, residual: bool = False):
    """(o, lse) of attention over packed sequences; see the module's text.

    Of the forward features, ``rescale_skip_threshold`` applies, and ``num_sms`` to all but
    small calls (those have one CTA per item); ``scheduler`` and ``cluster_mn`` do not.

    residual: also return what rounding o to bf16 took away, (o, lse, o_residual), for
    wan_flash_packed_bwd: its row sums of o * do are then free of that rounding, which
    shows in the gradients of rows with few keys."""
    k_offsets = q_offsets if k_offsets is None else k_offsets
    total_q, total_k, h, h_kv, n, device = _check(q, k, v, q_offsets, k_offsets)
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    q_offsets, k_offsets = q_offsets.contiguous(), k_offsets.contiguous()
    o = torch.empty_like(q)
    o_residual = torch.empty_like(q) if residual else None
    lse = q.new_empty((h, total_q), dtype=torch.float32)
    out = (o, lse, o_residual) if residual else (o, lse)
    if total_q == 0 or h == 0:
        return out
    size = _fwd_bytes(device.index, n, total_q, total_k, h)
    ws = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    f = features.get()
    _launch(_lib.lib().wf_packed_fwd_with, device, q.data_ptr(), k.data_ptr(), v.data_ptr(), q_offsets.data_ptr(),
            k_offsets.data_ptr(), o.data_ptr(), o_residual.data_ptr() if residual else None, lse.data_ptr(),
            ws.data_ptr() if size else None, size, n, total_q, total_k, h, h_kv, 1 if causal else 0,
            _fwd_cfg(f.rescale_skip_threshold, f.num_sms))
    return out


def wan_flash_packed_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
                         do: torch.Tensor, q_offsets: torch.Tensor, k_offsets: torch.Tensor | None = None,
                         causal: bool = False, o_residual: torch.Tensor | None = None):
    """(dq, dk, dv) given the forward's o and lse (and o_residual, if it made one) and
    the gradient of o.

    dk and dv are bitwise reproducible; dq is accumulated with fp32 reductions
    unless ``features.set_bwd_overrides(deterministic=True)``.  ``nsplit`` of the
    backward features cuts the longest key tile's walk into that many pieces (0:
    the device chooses), ``pdl=False`` launches the four kernels plainly; the CTA-pair form does
    not apply."""
    k_offsets = q_offsets if k_offsets is None else k_offsets
    total_q, total_k, h, h_kv, n, device = _check(q, k, v, q_offsets, k_offsets)
    assert o.dtype is torch.bfloat16 and do.dtype is torch.bfloat16 and o.shape == q.shape and do.shape == q.shape
    assert lse.dtype is torch.float32 and lse.shape == (h, total_q)
    assert o.device == device and lse.device == device and do.device == device, "tensors must be on one CUDA device"
    if o_residual is not None:
        assert o_residual.dtype is torch.bfloat16 and o_residual.shape == q.shape and o_residual.device == device
        o_residual = _aligned(o_residual)
    q, k, v, o, do, lse = _aligned(q), _aligned(k), _aligned(v), _aligned(o), _aligned(do), lse.contiguous()
    q_offsets, k_offsets = q_offsets.contiguous(), k_offsets.contiguous()
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    if total_q == 0 or total_k == 0 or h == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    f = features.get_bwd()
    cfg, size = _bwd_cfg_bytes(device.index, n, total_q, total_k, h, h_kv, f.nsplit, f.deterministic, f.pdl)
    ws = torch.empty(size, dtype=torch.uint8, device=device)
    _launch(_lib.lib().wf_packed_bwd_with, device, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
            None if o_residual is None else o_residual.data_ptr(), lse.data_ptr(), do.data_ptr(), q_offsets.data_ptr(),
            k_offsets.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
            ws.data_ptr(), size, n, total_q, total_k, h, h_kv, 1 if causal else 0, cfg)
    return dq, dk, dv


class _WanFlashAttnPackedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_offsets, k_offsets, causal):
        o, lse, o_residual = wan_flash_packed_fwd(q, k, v, q_offsets, k_offsets, causal, residual=True)
        ctx.save_for_backward(q, k, v, o, lse, o_residual, q_offsets, k_offsets)
        ctx.causal = causal
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        if _has_tangent(do):
            raise NotImplementedError("packed attention's backward has no forward-mode derivative")
        q, k, v, o, lse, o_residual, q_offsets, k_offsets = ctx.saved_tensors
        dq, dk, dv = wan_flash_packed_bwd(q, k, v, o, lse, do, q_offsets, k_offsets, ctx.causal, o_residual)
        return dq, dk, dv, None, None, None


def wan_flash_attn_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_offsets: torch.Tensor,
                          k_offsets: torch.Tensor | None = None, causal: bool = False):
    """Differentiable (once, in reverse mode) attention over packed sequences -> o (total_q, h, 128)
    bf16.  A tensor with a forward-mode tangent raises NotImplementedError, as wan_flash_attn does."""
    k_offsets = q_offsets if k_offsets is None else k_offsets
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) or _has_tangent(q, k, v):
        return _WanFlashAttnPackedFn.apply(q, k, v, q_offsets, k_offsets, bool(causal))
    return wan_flash_packed_fwd(q, k, v, q_offsets, k_offsets, causal)[0]
