"""Rotary positions: the table and the positions, the kernel against the
complex product in 64 bits, its gradients, strides, padding and refusals."""

import pytest
import torch

from wan_flash import _lib
from wan_flash.rope import AXES, rope_positions, rope_table, wan_flash_rope


def turned64(x, positions, theta=10000.0, axes=AXES, sign=1.0):
    """x (..., s, h, 128) times exp(i angle), angles from the definition in fp64."""
    f = [theta ** (-torch.arange(0, d, 2, dtype=torch.float64, device=x.device) / max(d, 1)) for d in axes]
    pos = positions.double()
    angle = torch.cat([pos[..., a:a + 1] * f[a] for a in range(3)], -1)
    angle = torch.where((positions < 0).any(-1, keepdim=True), 0.0, angle)[..., None, :]
    z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], 64, 2))
    return torch.view_as_real(z * torch.polar(torch.ones_like(angle), sign * angle)).flatten(-2)


def rope_tol(x, want):
    """One rounding of the result to x's type, and fp32 products of table entries
    that are half an fp32 step off: (2 * 2^-24 + 2^-24) of each of the pair's values."""
    pair = x.double().reshape(*x.shape[:-1], 64, 2).abs().sum(-1, keepdim=True).expand(*x.shape[:-1], 64, 2).flatten(-2)
    return torch.finfo(x.dtype).eps / 2 * want.abs() * (1 + 2**-7) + 4 * 2.0**-24 * pair


def test_table_and_positions():
    t = rope_table(50, theta=100.0, axes=(64, 0, 64))
    assert t.shape == (50, 64, 2) and t.dtype == torch.float32
    for p, i in ((0, 0), (49, 0), (49, 31), (7, 32), (33, 63)):
        angle = torch.tensor(p * 100.0 ** (-2 * (i % 32) / 64), dtype=torch.float64)
        assert abs(t[p, i, 0].item() - angle.cos().item()) <= 2**-24
        assert abs(t[p, i, 1].item() - angle.sin().item()) <= 2**-24
    pos = rope_positions((2, 3, 4))
    assert pos.dtype == torch.int32 and pos.tolist() == [[a, b, c] for a in range(2) for b in range(3) for c in range(4)]
    # a shard, a continued clip, and padding behind the grid
    assert rope_positions((2, 3, 4), start=22, count=4, first_frame=5).tolist() == [[6, 2, 2], [6, 2, 3], [-1] * 3, [-1] * 3]
    assert rope_positions((0, 3, 4)).shape == (0, 3)
    with pytest.raises(AssertionError):
        rope_table(10, axes=(64, 32, 31))
    with pytest.raises(AssertionError):
        rope_positions((1, 2, 3), start=-1)


def test_refusals():
    q, pos, table = torch.zeros(1, 4, 2, 128, dtype=torch.bfloat16), torch.zeros(4, 3, dtype=torch.int32), rope_table(8)
    for bad in (
        (q, q, pos, table),                                    # CPU tensors
        (q.half(), q.half(), pos, table),
        (q, q.float(), pos, table),
        (q[..., :64], q[..., :64], pos, table),
        (q, q[:, :3], pos, table),                             # another number of tokens
        (q, q, pos[:3], table),
        (q, q, pos.long(), table),
        (q, q, pos, table.double()),
        (q, q, pos, table[:, :32]),
        (q, q, pos, table[:0]),
        (q, q, pos, table, (44, 42, 40)),
    ):
        with pytest.raises(AssertionError):
            wan_flash_rope(*bad)


def test_c_entry_refusals():
    import ctypes

    lib = _lib.lib()

    def call(q=16, b=1, s=4, h=2, hk=2, null_cfg=False, **kw):
        cfg = _lib.RopeCfg(0, 0, 8, 22, 21, 0, 1024, 256, 128, 1024, 256, 128, 0)
        for k, v in kw.items():
            setattr(cfg, k, v)
        p = ctypes.c_void_p
        return lib.wf_rope(p(q) if q else None, p(32), p(48), p(64), p(80), p(96), b, s, h, hk,
                           None if null_cfg else ctypes.byref(cfg), None)

    assert call(s=-1) == -1 and call(null_cfg=True) == -1 and call(dtype=7) == -2 and call(max_pos=0) == -1
    assert call(pairs_t=60) == -1 and call(q=None) == -1 and call(h=70000) == -2
    assert call(q=24) == -3 and call(q_stride_s=250) == -3
    assert call(b=0) == 0 and call(s=0) == 0  # nothing to do


CASES = [
    # b, grid, pad, h, hk
    (1, (1, 1, 1), 0, 1, 1),
    (2, (3, 5, 7), 2, 3, 1),
    (1, (2, 30, 52), 0, 12, 12),
    (3, (1, 9, 11), 5, 40, 8),
    (1, (1, 3, 3), 0, 0, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,grid,pad,h,hk", CASES)
def test_forward_and_gradients(b, grid, pad, h, hk, dtype):
    n = grid[0] * grid[1] * grid[2]
    g = torch.Generator().manual_seed(n)
    table = rope_table(1024, device="cuda")
    pos = rope_positions(grid, count=n + pad, first_frame=900, device="cuda")
    x = [torch.randn(b, n + pad, hh, 128, generator=g).to("cuda", dtype) for hh in (h, hk, h, hk)]
    q, k = x[0].requires_grad_(), x[1].requires_grad_()
    yq, yk = wan_flash_rope(q, k, pos, table)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (x[2], x[3]))
    _lib.check_device()
    for src, got, sign in ((q, yq, 1), (k, yk, 1), (x[2], gq, -1), (x[3], gk, -1)):
        want = turned64(src.detach(), pos, sign=sign)
        assert got.dtype == dtype and got.is_contiguous() and got.shape == src.shape
        assert ((got.detach().double() - want).abs() <= rope_tol(src.detach(), want)).all()
    if pad:
        assert torch.equal(yq[:, n:], q[:, n:])  # padding passes bit for bit


@pytest.mark.gpu
def test_gradient_against_differences():
    table, pos = rope_table(64, device="cuda"), rope_positions((2, 2, 3), device="cuda")
    g = torch.Generator().manual_seed(3)
    q, k, w, dq = (torch.randn(12, 2, 128, generator=g).cuda() for _ in range(4))
    q.requires_grad_()
    loss = (wan_flash_rope(q, k, pos, table)[0] * w).sum()
    (grad,) = torch.autograd.grad(loss, q)
    # the map is linear: a central difference is exact but for rounding.  Each term
    # |w y| is off by a few fp32 steps of (|x0| + |x1|) |w|
    up = (wan_flash_rope(q.detach() + dq, k, pos, table)[0].double() * w.double()).sum()
    down = (wan_flash_rope(q.detach() - dq, k, pos, table)[0].double() * w.double()).sum()
    got, want = (grad.double() * dq.double()).sum().item(), ((up - down) / 2).item()
    tol = 8 * 2.0**-24 * 4 * ((q.detach().abs() + dq.abs()) * w.abs()).double().sum().item()
    assert abs(got - want) <= tol


@pytest.mark.gpu
def test_second_derivative():
    """The gradient is a turn itself: turning it on gives the identity's rounding error only."""
    table, pos = rope_table(64, device="cuda"), rope_positions((2, 2, 3), device="cuda")
    g = torch.Generator().manual_seed(4)
    q, k, w, x = (torch.randn(12, 2, 128, generator=g).cuda() for _ in range(4))
    q.requires_grad_(), w.requires_grad_()
    (grad,) = torch.autograd.grad((wan_flash_rope(q, k, pos, table)[0] * w).sum(), q, create_graph=True)
    (back,) = torch.autograd.grad((grad * x).sum(), w)  # d/dw of <turn^-1 w, x> = turn x
    want = turned64(x, pos)
    assert ((back.double() - want).abs() <= rope_tol(x, want)).all()


@pytest.mark.gpu
def test_strided_packed_and_per_item_positions():
    g = torch.Generator().manual_seed(5)
    table = rope_table(128, device="cuda")
    qkv = torch.randn(2, 10, 3, 4, 128, generator=g).to("cuda", torch.bfloat16)
    pos = torch.stack([rope_positions((1, 2, 5), device="cuda"), rope_positions((10, 1, 1), first_frame=7, device="cuda")])
    q, k = qkv[:, :, 0], qkv[:, :, 1]  # slices of a fused projection, read by their strides
    yq, yk = wan_flash_rope(q, k, pos, table)
    for src, got in ((q, yq), (k, yk)):
        want = turned64(src, pos)
        assert ((got.double() - want).abs() <= rope_tol(src, want)).all()
    # one packed sequence is the item without its batch dim; a misaligned or transposed view is copied
    a, b = wan_flash_rope(q[1], k[1], pos[1], table)
    assert torch.equal(a, yq[1]) and torch.equal(b, yk[1])
    flat = torch.zeros(2 * 10 * 4 * 128 + 1, device="cuda", dtype=torch.bfloat16)
    odd = flat[1:].view(2, 10, 4, 128).copy_(q)
    assert torch.equal(wan_flash_rope(odd, k, pos, table)[0], yq)
    swapped = q.transpose(1, 3).contiguous().transpose(1, 3)
    assert torch.equal(wan_flash_rope(swapped, k, pos, table)[0], yq)
    # heads broadcast from one
    one = q[:, :, :1].expand(2, 10, 4, 128)
    assert torch.equal(wan_flash_rope(one, k, pos, table)[0], yq[:, :, :1].expand(2, 10, 4, 128))
    _lib.check_device()


@pytest.mark.gpu
def test_strides_past_32_bits():
    table, pos = rope_table(64, device="cuda"), rope_positions((3, 2, 1), device="cuda")
    q, k = (torch.randn(6, 3, 128, device="cuda").bfloat16() for _ in range(2))
    want = wan_flash_rope(q, k, pos, table)
    big = torch.empty(5 * 2**29 + 6 * 128, dtype=torch.bfloat16, device="cuda")  # 5 GiB
    tokens = torch.as_strided(big, (6, 3, 128), (2**29, 128, 1)).copy_(q)
    heads = torch.as_strided(big, (6, 3, 128), (128, 2**30, 1), 3 * 128)
    got = wan_flash_rope(tokens, k, pos, table)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    heads.copy_(k)
    assert torch.equal(wan_flash_rope(q, heads, pos, table)[1], want[1])
    _lib.check_device()


@pytest.mark.gpu
def test_far_position_is_an_error_of_its_token_only():
    table = rope_table(16, device="cuda")
    pos = torch.tensor([[1, 2, 3], [1, 16, 3], [15, 15, 15]], dtype=torch.int32, device="cuda")
    q = torch.randn(3, 2, 128, device="cuda")
    y, _ = wan_flash_rope(q, q, pos, table)
    with pytest.raises(_lib.WanFlashError):
        _lib.check_device()
    assert y[1].isnan().all() and y[[0, 2]].isfinite().all()
    _lib.check_device()  # the read cleared it


@pytest.mark.gpu
def test_graph_replay_and_other_stream():
    table, pos = rope_table(64, device="cuda"), rope_positions((4, 4, 4), device="cuda")
    q, k = (torch.randn(64, 3, 128, device="cuda") for _ in range(2))
    want = wan_flash_rope(q, k, pos, table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = wan_flash_rope(q, k, pos, table)
        graph = torch.cuda.CUDAGraph()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            out = wan_flash_rope(q, k, pos, table)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], -want[0]) and torch.equal(out[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_behind_a_kernel_of_another_stream(captured):
    """The first kernel may come up early behind its own stream's last one, never before the stream it waits for."""
    table, pos = rope_table(64, device="cuda"), rope_positions((4, 4, 4), device="cuda")
    q, k = (torch.randn(64, 3, 128, device="cuda") for _ in range(2))

    def call(x):
        return wan_flash_rope(x, k, pos, table)

    want = call(q)
    late = torch.zeros_like(q)
    big = torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16)
    side = torch.cuda.Stream()

    def run():
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            late.copy_(q + (big @ big)[0, 0] * 0)  # a millisecond behind
        other = big[:64] * 2  # a short kernel of this stream
        here.wait_stream(side)
        out = call(late)
        return out, other

    run()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
    for _ in range(3):
        late.zero_()
        torch.cuda.synchronize()
        if captured:
            graph.replay()
        else:
            out = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out[0], want))
    _lib.check_device()


@pytest.mark.gpu
def test_right_behind_writers_of_its_inputs():
    """Each call reads what the kernels just before it wrote, also in place of older values."""
    g = torch.Generator().manual_seed(2)
    table = rope_table(64, device="cuda")
    src = torch.randn(40, 64, 3, 128, generator=g).to("cuda", torch.bfloat16)
    grids = [rope_positions((4, 4, 4), first_frame=i, device="cuda") for i in range(40)]
    x, pos, got = torch.empty_like(src[0]), torch.empty_like(grids[0]), []
    for i in range(40):
        torch.mul(src[i], 1, out=x)
        torch.add(grids[i], 0, out=pos)
        got.append(wan_flash_rope(x, x, pos, table)[0])
    for i in range(40):
        assert torch.equal(got[i], wan_flash_rope(src[i], src[i], grids[i], table)[0])
    _lib.check_device()


def _check_forward_mode(call, q, k, tq, tk):
    """The tangent of a turn is the turned tangent, with grad mode on or off, for
    leaves and plain tensors, for one tensor or both, and through the backward."""
    from torch.autograd import forward_ad

    want, zero = call(tq, tk), torch.zeros_like(k)
    for grad_mode in (False, True):
        for leaf in (False, True):
            with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
                x, y = (t.clone().requires_grad_(leaf) for t in (q, k))
                both = call(forward_ad.make_dual(x, tq), forward_ad.make_dual(y, tk))
                one = call(forward_ad.make_dual(x, tq), y)
                for out, t in zip((*both, *one), (*want, want[0], zero)):
                    got = forward_ad.unpack_dual(out).tangent
                    assert torch.equal(torch.zeros_like(t) if got is None and t is zero else got, t)
                assert all(torch.equal(a, b) for a, b in zip(both, call(q, k)))
    with forward_ad.dual_level():
        x = q.clone().requires_grad_()
        out, _ = call(x, k)
        (gq,) = torch.autograd.grad(out, x, forward_ad.make_dual(q, tq))
        back, _ = call(x, k)
        (plain,) = torch.autograd.grad(back, x, tq)
        assert torch.equal(forward_ad.unpack_dual(gq).tangent, plain)


@pytest.mark.parametrize("op", [False, True])
def test_forward_mode_derivative_on_a_stand_in(monkeypatch, op):
    from torch.autograd import forward_ad

    import wan_flash.rope
    import wan_flash.torch_op

    def launch(q, k, positions, table, axes, inverse):  # knows no derivative, like the kernel
        return tuple(turned64(forward_ad.unpack_dual(x.detach()).primal, positions, axes=axes, sign=-1.0 if inverse else 1.0)
                     for x in (q, k))

    for module in (wan_flash.rope, wan_flash.torch_op):
        monkeypatch.setattr(module, "_rope_impl", launch)
    g = torch.Generator().manual_seed(3)
    q, k, tq, tk = (torch.randn(24, h, 128, dtype=torch.float64, generator=g) for h in (3, 2, 3, 2))
    pos, table = rope_positions((2, 3, 4)), rope_table(8)
    fn = wan_flash.torch_op.wan_rope if op else wan_flash_rope
    _check_forward_mode(lambda a, b: fn(a, b, pos, table), q, k, tq, tk)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_forward_mode_derivative(dtype):
    from wan_flash.torch_op import wan_rope

    g = torch.Generator().manual_seed(3)
    q, k, tq, tk = (torch.randn(24, h, 128, generator=g).to("cuda", dtype) for h in (3, 2, 3, 2))
    pos, table = rope_positions((2, 3, 4), device="cuda"), rope_table(8, device="cuda")
    for fn in (wan_flash_rope, wan_rope):
        _check_forward_mode(lambda a, b: fn(a, b, pos, table), q, k, tq, tk)
    _lib.check_device()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("axes", [AXES, (64, 0, 64), (0, 64, 64), (64, 64, 0), (128, 0, 0), (0, 0, 128), (2, 62, 64)])
def test_other_splits_of_the_axes(axes, dtype):
    """Forward and gradients against the definition; a large coordinate on an axis without dims turns
    nothing, on another it is past the table."""
    g = torch.Generator().manual_seed(4)
    q, k, gq, gk = (torch.randn(24, h, 128, generator=g).to("cuda", dtype) for h in (3, 2, 3, 2))
    table, pos = rope_table(8, axes=axes, device="cuda"), rope_positions((2, 3, 4), first_frame=3, device="cuda")
    pos[5] = -1
    for a, d in enumerate(axes):
        if d == 0:
            pos[:5, a] = 2**31 - 1
    leaves = [x.clone().requires_grad_() for x in (q, k)]
    out = wan_flash_rope(*leaves, pos, table, axes)
    grads = torch.autograd.grad(out, leaves, (gq, gk))
    _lib.check_device()
    for got, x, sign in zip((*out, *grads), (q, k, gq, gk), (1.0, 1.0, -1.0, -1.0)):
        want = turned64(x, pos, axes=axes, sign=sign)
        assert ((got.double() - want).abs() <= rope_tol(x, want)).all()
    for a, d in enumerate(axes):
        if d > 0:
            bad = pos.clone()
            bad[7, a] = 8
            out = wan_flash_rope(q, k, bad, table, axes)
            with pytest.raises(_lib.WanFlashError):
                _lib.check_device()
            for x in out:
                assert x[7].isnan().all() and not x[:7].isnan().any() and not x[8:].isnan().any()
