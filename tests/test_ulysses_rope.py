"""Rotary positions in the sequence-parallel self attention: every rank turns its
shard with its own positions, and the result and gradients equal the
single-process computation (gloo ranks on the CPU, a CPU reference for the
turn and the attention; on the GPU, one NCCL rank with the kernels)."""

import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from tests.test_ulysses import _free_port, _ref_attn
from wan_flash.rope import rope_positions, rope_table

GRID = (2, 3, 4)


def _ref_rope(q, k, positions, table):
    def turned(x):
        at = positions.clamp(min=0).long()
        pair = torch.arange(64)
        cs = table[at[:, (pair >= 22).long() + (pair >= 43).long()], pair][:, None]  # (s, 1, 64, 2)
        z = torch.view_as_complex(x.reshape(*x.shape[:-1], 64, 2)) * torch.view_as_complex(cs.contiguous())
        return torch.view_as_real(z).flatten(-2)

    return turned(q), turned(k)


def _worker(rank, world, port, result_q):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from wan_flash import ulysses

        torch.manual_seed(0)
        S, n = 24, 24 // world
        q, k, v, g = (torch.randn(1, S, 4, 128) for _ in range(4))
        table = rope_table(16)
        full = [t.clone().requires_grad_() for t in (q, k, v)]
        want = _ref_attn(*_ref_rope(full[0], full[1], rope_positions(GRID), table), full[2])
        want.backward(g)
        rows = slice(rank * n, (rank + 1) * n)
        mine = [t[:, rows].clone().requires_grad_() for t in (q, k, v)]
        positions = rope_positions(GRID, start=rank * n, count=n)
        got = ulysses.ulysses_self_attention(*mine, attn_fn=_ref_attn, rope=(positions, table), rope_fn=_ref_rope)
        got.backward(g[:, rows])
        errs = [(got - want[:, rows]).abs().max().item()]
        errs += [(a.grad - b.grad[:, rows]).abs().max().item() for a, b in zip(mine, full)]
        result_q.put((rank, errs))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 4])
def test_ranks_turn_their_own_shards(world):
    ctx = mp.get_context("spawn")
    result_q, port = ctx.Queue(), _free_port()
    procs = [ctx.Process(target=_worker, args=(r, world, port, result_q)) for r in range(world)]
    for p in procs:
        p.start()
    got = [result_q.get(timeout=120) for _ in procs]
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    # sums of at most 24 fp32 products of values below 20, and two softmaxes in another order
    assert all(e <= 2e-4 for _, errs in got for e in errs), got


@pytest.mark.gpu
def test_one_rank_with_the_kernels():
    from wan_flash import _lib, ulysses
    from wan_flash.interface import wan_flash_attn
    from wan_flash.rope import wan_flash_rope

    dist.init_process_group("nccl", init_method=f"tcp://127.0.0.1:{_free_port()}", rank=0, world_size=1)
    try:
        g = torch.Generator().manual_seed(1)
        q, k, v = (torch.randn(1, 24, 2, 128, generator=g).to("cuda", torch.bfloat16) for _ in range(3))
        rope = rope_positions(GRID, device="cuda"), rope_table(16, device="cuda")
        got = ulysses.ulysses_self_attention(q, k, v, rope=rope)
        assert torch.equal(got, wan_flash_attn(*wan_flash_rope(q, k, *rope), v))
        assert not torch.equal(got, ulysses.ulysses_self_attention(q, k, v))
        _lib.check_device()
    finally:
        dist.destroy_process_group()
