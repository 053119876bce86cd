"""Rotary positions, packed attention and decode as torch.library ops: fakes with
the contract's shapes and strides (CPU), the kernels' own results, autograd,
activation checkpointing and torch.compile (GPU)."""

import pytest
import torch

import wan_flash.torch_op as op
from wan_flash.rope import rope_positions, rope_table


def test_fakes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    def t(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    with FakeTensorMode():
        q, k = t(50, 4, 128).transpose(0, 1).contiguous().transpose(0, 1), t(60, 2, 128)
        off = t(4, dtype=torch.int32)
        o, lse, res = torch.ops.wan_flash.packed_fwd(q, k, k, off, off, True)
        assert o.shape == res.shape == q.shape and o.is_contiguous() and lse.shape == (4, 50) and lse.dtype == torch.float32
        grads = torch.ops.wan_flash.packed_bwd(q, k, k, o, lse, res, o, off, off, True)
        assert [g.shape for g in grads] == [q.shape, k.shape, k.shape] and all(g.is_contiguous() for g in grads)
        a, b = op.wan_rope(q, t(50, 2, 128), t(50, 3, dtype=torch.int32), t(16, 64, 2, dtype=torch.float32))
        assert a.shape == q.shape and a.is_contiguous() and b.shape == (50, 2, 128)
        o, lse = torch.ops.wan_flash.decode(t(3, 4, 128), t(9, 16, 2, 128), t(9, 16, 2, 128), t(3, 5, dtype=torch.int32),
                                            t(3, dtype=torch.int32))
        assert o.shape == (3, 4, 128) and lse.shape == (3, 4)
    leaves = [torch.empty(50, h, 128, dtype=torch.bfloat16, device="meta", requires_grad=True) for h in (4, 2, 2)]
    off = torch.empty(4, dtype=torch.int32, device="meta")
    out = op.wan_attention_packed(*leaves, off, causal=True)
    out.backward(torch.empty_like(out))
    assert all(x.grad.shape == x.shape for x in leaves)


def _step(leaves, pos, table, off, attend, rope):
    q, k = rope(leaves[0], leaves[1], pos, table)
    return attend(q, k, leaves[2], off, causal=True)


@pytest.mark.gpu
def test_ops_match_the_functions_and_trace():
    from torch.utils.checkpoint import checkpoint

    from tests.test_packed import make
    from wan_flash.packed import wan_flash_attn_packed
    from wan_flash.rope import wan_flash_rope

    q, k, v, do, off, _ = make([100, 37, 160], [100, 37, 160], 4, 2)
    pos = torch.cat([rope_positions(g, device="cuda") for g in ((1, 10, 10), (37, 1, 1), (2, 8, 10))])
    table = rope_table(64, device="cuda")

    def run(fn):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out = fn(leaves)
        return out.detach(), *torch.autograd.grad(out, leaves, do)

    want = run(lambda x: _step(x, pos, table, off, wan_flash_attn_packed, wan_flash_rope))
    by_ops = lambda x: _step(x, pos, table, off, op.wan_attention_packed, op.wan_rope)  # noqa: E731
    for fn in (by_ops, lambda x: checkpoint(by_ops, x, use_reentrant=False), torch.compile(by_ops, backend="aot_eager")):
        got = run(fn)
        assert torch.equal(got[0], want[0])
        for a, b in zip(got[1:], want[1:]):  # dq is summed in another order
            assert torch.allclose(a.float(), b.float(), rtol=2.0**-7, atol=2.0**-7)
    args = (q, k, v, off, off, True)
    torch.library.opcheck(torch.ops.wan_flash.packed_fwd.default, args, test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.wan_flash.rope.default, (q, k, pos, table, [44, 42, 42], False),
                          test_utils=("test_schema", "test_faketensor"))


@pytest.mark.gpu
def test_decode_op():
    from tests.test_decode import make
    from wan_flash.decode import wan_flash_decode

    args = make([40, 0, 7], 4, 2, 8)
    o, lse = torch.ops.wan_flash.decode(*args)
    want = wan_flash_decode(*args)
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1]) and torch.equal(op.wan_decode(*args), o)
    # unread page-table entries are out of range on purpose: opcheck clones, which is fine
    torch.library.opcheck(torch.ops.wan_flash.decode.default, args, test_utils=("test_schema", "test_faketensor"))


def test_residual_is_made_for_gradients_only(monkeypatch):
    """wan_attention_packed asks for o's rounding residual only where a gradient will read it, and the
    operator's backward works without one too."""
    asked, given = [], []

    def fwd(q, k, v, q_offsets, k_offsets, causal, residual=False):
        asked.append(residual)
        lse = torch.zeros(q.shape[1], q.shape[0])
        return (torch.zeros_like(q), lse, torch.zeros_like(q)) if residual else (torch.zeros_like(q), lse)

    def bwd(q, k, v, o, lse, do, q_offsets, k_offsets, causal, o_residual=None):
        given.append(o_residual)
        return torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)

    monkeypatch.setattr(op, "wan_flash_packed_fwd", fwd)
    monkeypatch.setattr(op, "wan_flash_packed_bwd", bwd)
    q, k = torch.zeros(8, 4, 128, dtype=torch.bfloat16), torch.zeros(8, 2, 128, dtype=torch.bfloat16)
    off = torch.tensor([0, 5, 8], dtype=torch.int32)
    op.wan_attention_packed(q, k, k, off)
    leaf = k.clone().requires_grad_()
    with torch.no_grad():
        op.wan_attention_packed(q, leaf, k, off)
    assert asked == [False, False]
    o = op.wan_attention_packed(q, leaf, k, off)
    torch.autograd.grad(o, leaf, o)
    assert asked == [False, False, True] and given[0].shape == q.shape
    o, _, res = torch.ops.wan_flash.packed_fwd(q, leaf, k, off, off, False, False)
    torch.autograd.grad(o, leaf, o)
    assert res.numel() == 0 and given[1] is None


@pytest.mark.gpu
def test_ops_without_a_residual():
    from tests.test_packed import make
    from wan_flash.packed import wan_flash_packed_bwd, wan_flash_packed_fwd

    q, k, v, do, off, _ = make([100, 37, 160], [100, 37, 160], 4, 2)
    o, lse = wan_flash_packed_fwd(q, k, v, off, causal=True)
    assert torch.equal(op.wan_attention_packed(q, k, v, off, causal=True), o)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    got = torch.ops.wan_flash.packed_fwd(*leaves, off, off, True, False)
    assert torch.equal(got[0], o) and torch.equal(got[1], lse)
    want = wan_flash_packed_bwd(q, k, v, o, lse, do, off, causal=True)
    grads = torch.autograd.grad(got[0], leaves, do)
    assert torch.equal(grads[1], want[1]) and torch.equal(grads[2], want[2])
    torch.library.opcheck(torch.ops.wan_flash.packed_fwd.default, (q, k, v, off, off, True, False),
                          test_utils=("test_schema", "test_faketensor"))
    compiled = torch.compile(lambda *x: op.wan_attention_packed(*x, off, causal=True), backend="aot_eager")
    with torch.no_grad():
        assert torch.equal(compiled(q, k, v), o)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(compiled(*leaves), leaves, do)
    direct = torch.autograd.grad(op.wan_attention_packed(*leaves, off, causal=True), leaves, do)
    assert torch.equal(grads[1], direct[1]) and torch.equal(grads[2], direct[2])
