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
position past the table, on an axis that has dims, is found on the device: its
token's rows become NaN and ``wan_flash._lib.check_device()`` raises.
"""

from __future__ import annotations

import functools

import torch

from wan_flash import _lib
from wan_flash.interface import _contiguous_like, _has_tangent, _launch
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


def _rows(x: torch.Tensor, size: int):
    """x itself where the kernel can read it by its strides (16-byte rows), else a
    contiguous copy; and its (batch, token, head) strides."""
    st = x.stride()
    batch = st[0] if len(st) == 4 else 0
    if st[-1] != 1 or (batch | st[-3] | st[-2]) % (16 // size) or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        st = x.stride()
        batch = st[0] if len(st) == 4 else 0
    return x, batch, st[-3], st[-2]


@functools.lru_cache(maxsize=256)
def _cfg(*sizes):
    """The C options of a shape and its strides (1.2 us to make, 0.2 to find)."""
    return _lib.RopeCfg(*sizes)


def _axes_ok(axes) -> bool:
    return len(axes) == 3 and sum(axes) == HEAD_DIM and all(d >= 0 and d % 2 == 0 for d in axes)


def _rope_impl(q, k, positions, table, axes, inverse):
    dtype = q.dtype
    assert k.dtype is dtype and (dtype is torch.bfloat16 or dtype is torch.float32), "q and k are both bf16 or both fp32"
    qs, kshape, ps = q.shape, k.shape, positions.shape
    dims = len(qs)
    assert len(kshape) == dims and (dims == 3 or dims == 4), "(s, h, 128) or (b, s, h, 128)"
    s, h, d = qs[-3:]
    ks, h_kv, dk = kshape[-3:]
    b = qs[0] if dims == 4 else 1
    assert ks == s and (dims == 3 or kshape[0] == b), "q and k have the same tokens"
    assert d == HEAD_DIM and dk == HEAD_DIM, "specialized for head_dim=128"
    assert axes is AXES or _axes_ok(axes), "three even axes that add up to head_dim"
    assert positions.dtype is torch.int32 and (ps == (s, 3) or (dims == 4 and ps == (b, s, 3))), \
        "positions are int32 (s, 3) or one (s, 3) per batch item"
    assert table.dtype is torch.float32 and table.dim() == 3 and table.shape[1:] == (HEAD_DIM // 2, 2)
    rows = table.shape[0]
    assert rows >= 1
    device = q.device
    assert q.is_cuda and k.device == device and positions.device == device and table.device == device, \
        "tensors must be on one CUDA device"
    size = 2 if dtype is torch.bfloat16 else 4
    q, q0, q1, q2 = _rows(q, size)
    k, k0, k1, k2 = _rows(k, size)
    oq, ok = _contiguous_like(q), _contiguous_like(k)
    if b == 0 or s == 0 or h + h_kv == 0:
        return oq, ok
    positions = positions.contiguous()
    if not table.is_contiguous() or table.data_ptr() % 16:
        table = table.clone(memory_format=torch.contiguous_format)
    cfg = _cfg(0 if size == 2 else 1, 1 if inverse else 0, rows, axes[0] // 2, axes[1] // 2, 0,
               q0, q1, q2, k0, k1, k2, 3 * s if len(ps) == 3 else 0)
    _launch(_lib.lib().wf_rope, device, q.data_ptr(), k.data_ptr(), oq.data_ptr(), ok.data_ptr(), table.data_ptr(),
            positions.data_ptr(), b, s, h, h_kv, cfg)
    return oq, ok


class _WanFlashRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, table, axes, inverse):
        ctx.save_for_backward(positions, table)
        ctx.save_for_forward(positions, table)
        ctx.axes, ctx.inverse = axes, inverse
        return _rope_impl(q, k, positions, table, axes, inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        positions, table = ctx.saved_tensors
        gq, gk = _turned(gq, gk, positions, table, ctx.axes, not ctx.inverse)
        return gq, gk, None, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        return _turned(tq, tk, *ctx.saved_tensors, ctx.axes, ctx.inverse)  # the turn is linear


def _turned(q, k, positions, table, axes, inverse):
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad)) or _has_tangent(q, k):
        return _WanFlashRopeFn.apply(q, k, positions, table, axes, inverse)
    return _rope_impl(q, k, positions, table, axes, inverse)


def wan_flash_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, axes=AXES):
    """q (b, s, h, 128) and k (b, s, h_kv, 128), or packed (s, h, 128) and
    (s, h_kv, 128), bf16 or fp32 -> their turned copies (contiguous).

    positions: int32 (s, 3), or (b, s, 3) for a grid of its own per batch item;
    a token with a negative position is padding and passes unchanged.
    table: rope_table(...), more rows than the largest position.
    axes: head dims of time, height, width, as given to rope_table.
    q and k may be strided views (slices of a fused qkv projection); heads may
    differ.  Differentiable in q and k (the turn by the negative angle), any number of times,
    in reverse and in forward mode."""
    return _turned(q, k, positions, table, axes, False)
