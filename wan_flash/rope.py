"""Rotary positions with three axes (time, height, width) for q and k.

The Wan models turn q and k by rotary positions right before the self
attention of this package: of the 64 dim pairs of a 128-dim head, 22 follow
the token's frame, 21 its row and 21 its column.  The reference package
leaves that to the caller (complex128 torch code); here it is one kernel over
q and k.

rope_table(max_pos, ...) -> table        (max_pos, 64, 2) fp32: cos and sin
rope_positions(grid, ...) -> positions   (s, 3) int32 of a t x h x w grid
wan_flash_rope(q, k, positions, table) -> (q_rot, k_rot)   differentiable

Make the table once and the positions once per grid and keep them, as the
model keeps its frequency table.  Contract violations raise AssertionError
before any CUDA call; the kernel runs on ``torch.cuda.current_stream()``.  A
position past the table is found on the device: its token's rows become NaN
and ``wan_flash._lib.check_device()`` raises.
"""

from __future__ import annotations

import ctypes

import torch

from wan_flash import _lib
from wan_flash.interface import _ptr, _stream_ptr
from wan_flash.shapes import HEAD_DIM

AXES = (44, 42, 42)  # head dims of time, height, width in the Wan models


def rope_table(max_pos: int = 1024, theta: float = 10000.0, axes=AXES, device=None) -> torch.Tensor:
    """(max_pos, 64, 2) fp32 of (cos, sin): row p, pair i (the j-th of axis a,
    which holds axes[a] dims) is the angle p * theta^(-2j / axes[a]), computed
    in fp64."""
    assert sum(axes) == HEAD_DIM and len(axes) == 3 and all(d >= 0 and d % 2 == 0 for d in axes), \
        "three even axes that add up to head_dim"
    assert max_pos >= 1
    freq = torch.cat([theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / max(d, 1)) for d in axes])
    angle = torch.arange(max_pos, dtype=torch.float64)[:, None] * freq
    return torch.stack((angle.cos(), angle.sin()), -1).float().to(device or "cpu")


def rope_positions(grid, start: int = 0, count: int | None = None, first_frame: int = 0, device=None) -> torch.Tensor:
    """(count, 3) int32 positions (frame, row, column) of tokens [start, start + count)
    of a (t, h, w) grid in row-major order (all tokens by default).  A
    sequence-parallel rank passes its shard's start; a clip that continues a
    video passes its first frame; tokens behind the grid are padding (-1)."""
    t, h, w = (int(x) for x in grid)
    assert t >= 0 and h >= 0 and w >= 0 and start >= 0 and first_frame >= 0
    n = t * h * w
    count = n - start if count is None else count
    assert count >= 0
    i = torch.arange(start, start + count, device=device)
    hw, ww = max(h * w, 1), max(w, 1)
    pos = torch.stack((first_frame + i // hw, i // ww % max(h, 1), i % ww), 1)
    return torch.where((i < n)[:, None], pos, -1).to(torch.int32)


def _in_place(x: torch.Tensor) -> torch.Tensor:
    """x itself where the kernel can read it by its strides (16-byte rows), else a contiguous copy."""
    per16 = 16 // x.element_size()
    if x.stride(-1) == 1 and all(s % per16 == 0 and s >= 0 for s in x.stride()[:-1]) and x.data_ptr() % 16 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _rope_impl(q, k, positions, table, axes, inverse):
    assert q.dtype == k.dtype and q.dtype in (torch.bfloat16, torch.float32), "q and k are both bf16 or both fp32"
    assert q.dim() == k.dim() and q.dim() in (3, 4), "(s, h, 128) or (b, s, h, 128)"
    assert q.shape[:-2] == k.shape[:-2] and q.shape[-1] == k.shape[-1]
    assert q.shape[-1] == HEAD_DIM, "specialized for head_dim=128"
    assert len(axes) == 3 and sum(axes) == HEAD_DIM and all(d >= 0 and d % 2 == 0 for d in axes), \
        "three even axes that add up to head_dim"
    s = q.shape[-3]
    assert positions.dtype == torch.int32 and positions.shape[-1:] == (3,)
    assert positions.shape in ((s, 3), tuple(q.shape[:-2]) + (3,)), "positions are (s, 3) or one (s, 3) per batch item"
    assert table.dtype == torch.float32 and table.dim() == 3 and table.shape[1:] == (HEAD_DIM // 2, 2)
    assert table.shape[0] >= 1
    assert q.is_cuda and all(t.device == q.device for t in (k, positions, table)), "tensors must be on one CUDA device"
    b = q.shape[0] if q.dim() == 4 else 1
    oq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ok = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    if oq.numel() + ok.numel() == 0:
        return oq, ok
    q, k = _in_place(q), _in_place(k)
    positions = positions if positions.is_contiguous() else positions.contiguous()
    table = table if table.is_contiguous() and table.data_ptr() % 8 == 0 else table.clone(
        memory_format=torch.contiguous_format)
    st = [x.stride() if x.dim() == 4 else (0, *x.stride()) for x in (q, k)]
    cfg = _lib.RopeCfg(1 if q.dtype == torch.float32 else 0, 1 if inverse else 0, table.shape[0], axes[0] // 2,
                       axes[1] // 2, 0, st[0][0], st[0][1], st[0][2], st[1][0], st[1][1], st[1][2],
                       3 * s if positions.dim() == 3 else 0)
    with torch.cuda.device(q.device):
        rc = _lib.lib().wf_rope(_ptr(q), _ptr(k), _ptr(oq), _ptr(ok), _ptr(table), _ptr(positions), b, s, q.shape[-2],
                                k.shape[-2], ctypes.byref(cfg), ctypes.c_void_p(_stream_ptr(q.device)))
    _lib.check(rc)
    return oq, ok


class _WanFlashRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, table, axes):
        ctx.save_for_backward(positions, table)
        ctx.axes = axes
        return _rope_impl(q, k, positions, table, axes, False)

    @staticmethod
    def backward(ctx, gq, gk):
        positions, table = ctx.saved_tensors
        gq, gk = _rope_impl(gq, gk, positions, table, ctx.axes, True)
        return gq, gk, None, None, None


def wan_flash_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, axes=AXES):
    """q (b, s, h, 128) and k (b, s, h_kv, 128), or packed (s, h, 128) and
    (s, h_kv, 128), bf16 or fp32 -> their turned copies (contiguous).

    positions: int32 (s, 3), or (b, s, 3) for a grid of its own per batch item;
    a token with a negative position is padding and passes unchanged.
    table: rope_table(...), more rows than the largest position.
    axes: head dims of time, height, width, as given to rope_table.
    q and k may be strided views (slices of a fused qkv projection); heads may
    differ.  Differentiable in q and k (the turn by the negative angle)."""
    return _WanFlashRopeFn.apply(q, k, positions, table, tuple(int(d) for d in axes))
