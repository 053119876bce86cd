"""The attention as ``torch.library`` custom ops, for callers that trace.

The reference exposes a ``torch.autograd.Function`` (``interface.py:199-215``);
its consumer, the external ``wan_attention`` op, wants a registered operator
with a fake (meta) implementation so that graphs holding it can be traced
with fake tensors (``torch.compile``, export, activation checkpointing
replays) without running the kernels.  This module registers

    wan_flash::attn_fwd(q, k, v) -> (o, lse)
    wan_flash::attn_bwd(q, k, v, o, lse, do) -> (dq, dk, dv)

with fake implementations that only produce the contract's shapes and
dtypes -- o like q (bf16), lse (b, h, sq) fp32, gradients like their inputs --
and ties them together with ``register_autograd``.  The real
implementations are ``wan_flash_fwd`` / ``wan_flash_bwd`` (the sm_100a
kernels); nothing here computes on the CPU.

``wan_attention(q, k, v) -> o`` is the op-based counterpart of
``wan_flash_attn``.  The two-context path (Wan I2V text + image cross
attention) has the same treatment:

    wan_flash::attn_fwd_dual(q, k0, v0, k1, v1) -> (o0, lse0, o1, lse1)
    wan_flash::attn_bwd_dual(q, k0, v0, k1, v1, o0, lse0, o1, lse1, do0, do1)
        -> (dq, dk0, dv0, dk1, dv1)

and ``wan_attention_dual(q, k0, v0, k1, v1) -> o0 + o1``.  So have rotary
positions, packed attention and decode:

    wan_flash::rope(q, k, positions, table, axes, inverse) -> (q_rot, k_rot)
    wan_flash::packed_fwd(q, k, v, q_offsets, k_offsets, causal, residual=True)
        -> (o, lse, o_residual)      (o_residual empty without residual)
    wan_flash::packed_bwd(q, k, v, o, lse, o_residual, do, q_offsets, k_offsets, causal)
        -> (dq, dk, dv)
    wan_flash::decode(q, k_cache, v_cache, page_table, lengths) -> (o, lse)

with ``wan_rope``, ``wan_attention_packed`` (differentiable) and ``wan_decode``.
The operators themselves know no forward mode; ``wan_rope`` and
``wan_attention_packed`` treat tangents as the functions do.
"""

from __future__ import annotations

import torch

from wan_flash.decode import wan_flash_decode
from wan_flash.interface import _has_tangent, wan_flash_bwd, wan_flash_bwd_dual, wan_flash_fwd, wan_flash_fwd_dual
from wan_flash.packed import wan_flash_attn_packed, wan_flash_packed_bwd, wan_flash_packed_fwd
from wan_flash.rope import AXES, _rope_impl, _turned, wan_flash_rope


@torch.library.custom_op("wan_flash::attn_fwd", mutates_args=())
def attn_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    o, lse = wan_flash_fwd(q, k, v)
    return o, lse


def _like(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape, dtype and device: the real ops write
    contiguous (b, s, h, 128) outputs whatever the inputs' strides, so the fake
    outputs must not inherit a permuted input's strides."""
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


@attn_fwd.register_fake
def _attn_fwd_fake(q, k, v):
    b, sq, h, d = q.shape
    torch._check(d == 128, lambda: "specialized for head_dim=128")
    return _like(q), q.new_empty((b, h, sq), dtype=torch.float32)


@torch.library.custom_op("wan_flash::attn_bwd", mutates_args=())
def attn_bwd(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor, do: torch.Tensor
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    dq, dk, dv = wan_flash_bwd(q, k, v, o, lse, do)
    return dq, dk, dv


@attn_bwd.register_fake
def _attn_bwd_fake(q, k, v, o, lse, do):
    return _like(q), _like(k), _like(v)


def _setup_context(ctx, inputs, output):
    q, k, v = inputs
    o, lse = output
    # The LSE output carries no gradient (the reference's autograd function
    # returns o only): it is marked non-differentiable, so a loss that uses
    # it gets no gradient through it instead of a silently wrong one.
    ctx.mark_non_differentiable(lse)
    ctx.save_for_backward(q, k, v, o, lse)


def _backward(ctx, do, dlse):
    q, k, v, o, lse = ctx.saved_tensors
    dq, dk, dv = attn_bwd(q, k, v, o, lse, do.contiguous())
    return dq, dk, dv


attn_fwd.register_autograd(_backward, setup_context=_setup_context)


def wan_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """o = softmax(q k^T / sqrt(128)) v through the registered operator (differentiable)."""
    return attn_fwd(q, k, v)[0]


@torch.library.custom_op("wan_flash::attn_fwd_dual", mutates_args=())
def attn_fwd_dual(q: torch.Tensor, k0: torch.Tensor, v0: torch.Tensor, k1: torch.Tensor,
                  v1: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    o0, lse0, o1, lse1 = wan_flash_fwd_dual(q, k0, v0, k1, v1)
    return o0, lse0, o1, lse1


@attn_fwd_dual.register_fake
def _attn_fwd_dual_fake(q, k0, v0, k1, v1):
    b, sq, h, d = q.shape
    torch._check(d == 128, lambda: "specialized for head_dim=128")
    return _like(q), q.new_empty((b, h, sq), dtype=torch.float32), _like(q), q.new_empty((b, h, sq), dtype=torch.float32)


@torch.library.custom_op("wan_flash::attn_bwd_dual", mutates_args=())
def attn_bwd_dual(
    q: torch.Tensor, k0: torch.Tensor, v0: torch.Tensor, k1: torch.Tensor, v1: torch.Tensor, o0: torch.Tensor,
    lse0: torch.Tensor, o1: torch.Tensor, lse1: torch.Tensor, do0: torch.Tensor, do1: torch.Tensor
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return wan_flash_bwd_dual(q, k0, v0, k1, v1, o0, lse0, o1, lse1, do0, do1)


@attn_bwd_dual.register_fake
def _attn_bwd_dual_fake(q, k0, v0, k1, v1, o0, lse0, o1, lse1, do0, do1):
    return _like(q), _like(k0), _like(v0), _like(k1), _like(v1)


def _setup_context_dual(ctx, inputs, output):
    o0, lse0, o1, lse1 = output
    ctx.mark_non_differentiable(lse0, lse1)  # as in the one-context op
    ctx.save_for_backward(*inputs, o0, lse0, o1, lse1)


def _backward_dual(ctx, do0, dlse0, do1, dlse1):
    q, k0, v0, k1, v1, o0, lse0, o1, lse1 = ctx.saved_tensors
    return attn_bwd_dual(q, k0, v0, k1, v1, o0, lse0, o1, lse1, do0.contiguous(), do1.contiguous())


attn_fwd_dual.register_autograd(_backward_dual, setup_context=_setup_context_dual)


def wan_attention_dual(q: torch.Tensor, k0: torch.Tensor, v0: torch.Tensor, k1: torch.Tensor,
                       v1: torch.Tensor) -> torch.Tensor:
    """attention(q, k0, v0) + attention(q, k1, v1) through the registered operators (differentiable)."""
    o0, _, o1, _ = attn_fwd_dual(q, k0, v0, k1, v1)
    return o0 + o1


@torch.library.custom_op("wan_flash::rope", mutates_args=())
def rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, axes: list[int],
         inverse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return _rope_impl(q, k, positions, table, axes, inverse)


@rope.register_fake
def _rope_fake(q, k, positions, table, axes, inverse):
    torch._check(q.shape[-1] == 128, lambda: "specialized for head_dim=128")
    return _like(q), _like(k)


def _setup_context_rope(ctx, inputs, output):
    _, _, positions, table, axes, inverse = inputs
    ctx.save_for_backward(positions, table)
    ctx.axes, ctx.inverse = axes, inverse


def _backward_rope(ctx, gq, gk):
    turn = _turned if _has_tangent(gq, gk) else rope
    gq, gk = turn(gq, gk, *ctx.saved_tensors, ctx.axes, not ctx.inverse)
    return gq, gk, None, None, None, None


rope.register_autograd(_backward_rope, setup_context=_setup_context_rope)


def wan_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, axes=AXES):
    """wan_flash_rope through the registered operator (differentiable)."""
    if _has_tangent(q, k):  # an operator would drop it
        return wan_flash_rope(q, k, positions, table, axes)
    return rope(q, k, positions, table, list(axes), False)


@torch.library.custom_op("wan_flash::packed_fwd", mutates_args=())
def packed_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_offsets: torch.Tensor, k_offsets: torch.Tensor,
               causal: bool, residual: bool = True) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    out = wan_flash_packed_fwd(q, k, v, q_offsets, k_offsets, causal, residual=residual)
    return out if residual else (*out, q.new_empty(0))


@packed_fwd.register_fake
def _packed_fwd_fake(q, k, v, q_offsets, k_offsets, causal, residual=True):
    total_q, h, d = q.shape
    torch._check(d == 128, lambda: "specialized for head_dim=128")
    return _like(q), q.new_empty((h, total_q), dtype=torch.float32), _like(q) if residual else q.new_empty(0)


@torch.library.custom_op("wan_flash::packed_bwd", mutates_args=())
def packed_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
               o_residual: torch.Tensor, do: torch.Tensor, q_offsets: torch.Tensor, k_offsets: torch.Tensor,
               causal: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    given = o_residual.dim() == 3  # a forward without residual left an empty one
    return wan_flash_packed_bwd(q, k, v, o, lse, do, q_offsets, k_offsets, causal, o_residual if given else None)


@packed_bwd.register_fake
def _packed_bwd_fake(q, k, v, o, lse, o_residual, do, q_offsets, k_offsets, causal):
    return _like(q), _like(k), _like(v)


def _setup_context_packed(ctx, inputs, output):
    q, k, v, q_offsets, k_offsets, causal, _ = inputs
    o, lse, o_residual = output
    ctx.mark_non_differentiable(lse, o_residual)  # as in the dense op
    ctx.save_for_backward(q, k, v, o, lse, o_residual, q_offsets, k_offsets)
    ctx.causal = causal


def _backward_packed(ctx, do, dlse, dres):
    if _has_tangent(do):
        raise NotImplementedError("packed attention's backward has no forward-mode derivative")
    q, k, v, o, lse, o_residual, q_offsets, k_offsets = ctx.saved_tensors
    grads = packed_bwd(q, k, v, o, lse, o_residual, do.contiguous(), q_offsets, k_offsets, ctx.causal)
    return *grads, None, None, None, None


packed_fwd.register_autograd(_backward_packed, setup_context=_setup_context_packed)


def wan_attention_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_offsets: torch.Tensor,
                         k_offsets: torch.Tensor | None = None, causal: bool = False) -> torch.Tensor:
    """wan_flash_attn_packed through the registered operator (differentiable)."""
    if _has_tangent(q, k, v):  # an operator would drop it; this raises
        return wan_flash_attn_packed(q, k, v, q_offsets, k_offsets, causal)
    residual = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    return packed_fwd(q, k, v, q_offsets, q_offsets if k_offsets is None else k_offsets, causal, residual)[0]


@torch.library.custom_op("wan_flash::decode", mutates_args=())
def decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
           lengths: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return wan_flash_decode(q, k_cache, v_cache, page_table, lengths)


@decode.register_fake
def _decode_fake(q, k_cache, v_cache, page_table, lengths):
    b, h, d = q.shape
    torch._check(d == 128, lambda: "specialized for head_dim=128")
    return _like(q), q.new_empty((b, h), dtype=torch.float32)


def wan_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
               lengths: torch.Tensor) -> torch.Tensor:
    """o of wan_flash_decode through the registered operator."""
    return decode(q, k_cache, v_cache, page_table, lengths)[0]
