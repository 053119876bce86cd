"""The operators as an autoregressive video model uses them: rotary positions,
packed causal attention over the prompts, the paged cache, and decode steps,
against one causal attention over everything in 64 bits; and one training step
through rotary positions and packed attention against autograd in 64 bits."""

import pytest
import torch

from tests.attn64 import U, assert_close, attn64, grads64
from tests.test_packed import offsets
from tests.test_rope import rope_tol, turned64
from wan_flash import _lib
from wan_flash.decode import wan_flash_decode
from wan_flash.packed import wan_flash_attn_packed, wan_flash_packed_fwd
from wan_flash.rope import rope_positions, rope_table, wan_flash_rope

pytestmark = pytest.mark.gpu

H, HK, PAGE = 6, 2, 16


def _tokens(n, h, g):
    return torch.randn(n, h, 128, generator=g).to("cuda", torch.bfloat16)


def test_prompts_then_steps():
    """Two clips of other grids: prompts in one packed call, then their tokens one by one."""
    g = torch.Generator().manual_seed(0)
    grids, prompt = [(3, 5, 9), (2, 4, 7)], [100, 41]  # 135 and 56 tokens, the prompts end inside a frame
    total = [t * h * w for t, h, w in grids]
    table = rope_table(32, device="cuda")
    pos = [rope_positions(x, device="cuda") for x in grids]
    q, k, v = ([_tokens(n, h, g) for n in total] for h in (H, HK, HK))
    turned = [wan_flash_rope(a, b, p, table) for a, b, p in zip(q, k, pos)]  # what the reference sees

    # prompts: packed
    off = offsets(prompt)
    pq, pk, pv = (torch.cat([x[:n] for x, n in zip(y, prompt)]) for y in (q, k, v))
    pq, pk = wan_flash_rope(pq, pk, torch.cat([x[:n] for x, n in zip(pos, prompt)]), table)
    o, _ = wan_flash_packed_fwd(pq, pk, pv, off, causal=True)
    got = [[o[:prompt[0]]], [o[prompt[0]:]]]

    # the cache: pages handed out in turn, written token by token
    pages = torch.arange(40, dtype=torch.int32, device="cuda").flip(0)[:24].reshape(2, 12).contiguous()
    k_cache, v_cache = (torch.full((40, PAGE, HK, 128), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(2))

    def write(i, first, kk, vv):
        at = torch.arange(first, first + kk.shape[0], device="cuda")
        k_cache[pages[i, at // PAGE].long(), at % PAGE] = kk
        v_cache[pages[i, at // PAGE].long(), at % PAGE] = vv

    for i in range(2):
        a = off.tolist()
        write(i, 0, pk[a[i]:a[i + 1]], pv[a[i]:a[i + 1]])

    # steps: both streams until the shorter one ends, then one
    for step in range(max(n - p for n, p in zip(total, prompt))):
        live = [i for i in range(2) if prompt[i] + step < total[i]]
        at = [prompt[i] + step for i in live]
        nq, nk = wan_flash_rope(torch.stack([q[i][t] for i, t in zip(live, at)])[:, None],
                                torch.stack([k[i][t] for i, t in zip(live, at)])[:, None],
                                torch.stack([pos[i][t:t + 1] for i, t in zip(live, at)]), table)
        for j, (i, t) in enumerate(zip(live, at)):
            write(i, t, nk[j], v[i][t:t + 1])
        lengths = torch.tensor([t + 1 for t in at], dtype=torch.int32, device="cuda")
        o, _ = wan_flash_decode(nq[:, 0], k_cache, v_cache, pages[live], lengths)
        for j, i in enumerate(live):
            got[i].append(o[j:j + 1])
    _lib.check_device()
    for i in range(2):
        r = attn64(turned[i][0], turned[i][1], v[i], causal=True)
        assert_close(torch.cat(got[i]), r["o"], r["o_tol"], f"stream {i}")


def test_training_step():
    """dq and dk come back through the turn: the kernel's packed gradient is within its bounds of
    the 64-bit gradient at the turned values, and turning it back adds one rounding."""
    g = torch.Generator().manual_seed(1)
    grids = [(1, 7, 9), (4, 3, 11)]
    lens = [t * h * w for t, h, w in grids]
    off, table = offsets(lens), rope_table(16, device="cuda")
    pos = torch.cat([rope_positions(x, device="cuda") for x in grids])
    q, k, v, do = (_tokens(sum(lens), h, g) for h in (H, HK, HK, H))
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    out = wan_flash_attn_packed(*wan_flash_rope(leaves[0], leaves[1], pos, table), leaves[2], off, causal=True)
    dq, dk, dv = torch.autograd.grad(out, leaves, do)
    _lib.check_device()
    tq, tk = wan_flash_rope(q, k, pos, table)
    first = 0
    for n in lens:
        s = slice(first, first + n)
        first += n
        want = grads64(tq[s], tk[s], v[s], do[s], causal=True, residual=True)
        assert_close(dv[s], *want["dv"], "dv")
        for name, got in (("dq", dq), ("dk", dk)):
            w, tol = want[name]
            back = turned64(w, pos[s], sign=-1)
            # a turned error is at most the pair's two errors; then the rounding of the turn
            pair = tol.reshape(*tol.shape[:-1], 64, 2).sum(-1, keepdim=True).expand(*tol.shape[:-1], 64, 2).flatten(-2)
            assert_close(got[s], back, pair + U * (back.abs() + pair) + rope_tol(got[s], back), name)
