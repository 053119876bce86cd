"""Packed attention, forward: against attention in 64 bits sequence by
sequence, with lengths around the tiles, empty sequences and rows, NaN in rows
outside every sequence, grouped heads, graphs, streams and refusals."""

import ctypes

import pytest
import torch

from tests.attn64 import assert_close, attn64
from wan_flash import _lib
from wan_flash.packed import wan_flash_packed_fwd


def offsets(lens, lead=0, device="cuda"):
    at = [lead]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=device)


def make(lq, lk, h, hk, lead=0, tail=0, std=1.0, seed=0, device="cuda"):
    """q, k, v, do and the offsets; lead rows before and tail rows behind the sequences hold NaN."""
    g = torch.Generator().manual_seed(seed)
    shapes = ((sum(lq), h), (sum(lk), hk), (sum(lk), hk), (sum(lq), h))
    out = []
    for i, (n, hh) in enumerate(shapes):
        x = torch.randn(n, hh, 128, generator=g) * (std if i < 2 else 1.0)
        nan = torch.full((1, hh, 128), float("nan"))
        out.append(torch.cat((nan.expand(lead, -1, -1), x, nan.expand(tail, -1, -1))).to(device, torch.bfloat16))
    return (*out, offsets(lq, lead, device), offsets(lk, lead, device))


def check_fwd(q, k, v, qo, ko, causal, o, lse):
    qo, ko = qo.tolist(), ko.tolist()
    for i in range(len(qo) - 1):
        a, b, c, d = qo[i], qo[i + 1], ko[i], ko[i + 1]
        if a == b:
            continue
        r = attn64(q[a:b], k[c:d], v[c:d], causal)
        assert_close(o[a:b], r["o"], r["o_tol"], f"o of sequence {i}")
        assert_close(lse[:, a:b], r["lse"], r["lse_tol"], f"lse of sequence {i}")
    for rows in (slice(0, qo[0]), slice(qo[-1], None)):
        assert (o[rows] == 0).all() and (lse[:, rows] == float("-inf")).all()


CASES = [
    # lq, lk (None: the same), h, h_kv, causal
    ([1], None, 1, 1, True),
    ([1], None, 1, 1, False),
    ([128], None, 2, 1, True),
    ([129, 127, 256, 257, 255], None, 2, 2, True),
    ([129, 127, 256, 257, 255], None, 2, 2, False),
    ([64, 1, 0, 300, 0, 2], None, 3, 1, True),
    ([64, 1, 0, 300, 0, 2], None, 3, 1, False),
    ([5, 200, 128, 1], [133, 200, 400, 1000], 4, 2, True),     # continued prompts: more keys than queries
    ([5, 200, 128, 1], [133, 200, 400, 1000], 4, 2, False),
    ([300, 140, 7], [20, 0, 6], 2, 1, True),                   # fewer keys: rows that see nothing
    ([300, 140, 7], [20, 0, 6], 2, 1, False),
    ([0, 0], [10, 0], 2, 2, True),
    ([1111], None, 8, 1, True),
    ([700, 513], [130, 900], 12, 4, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk,h,hk,causal", CASES)
@pytest.mark.parametrize("lead,tail", [(0, 0), (3, 150)])
def test_forward(lq, lk, h, hk, causal, lead, tail):
    q, k, v, _, qo, ko = make(lq, lk or lq, h, hk, lead, tail)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal)
    _lib.check_device()
    assert o.shape == q.shape and o.dtype == torch.bfloat16 and lse.shape == (h, q.shape[0])
    check_fwd(q, k, v, qo, ko, causal, o, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk,lead,tail,causal", [
    ([300, 140, 1], None, 0, 40000, False),       # every SM has many tiles of padding behind its last with keys
    ([300, 140, 1], None, 40000, 0, True),
    ([300, 40000, 129], [300, 0, 257], 0, 0, False),
    ([40000, 77], [100, 77], 0, 0, True),         # most rows see no key
])
def test_many_tiles_without_keys(lq, lk, lead, tail, causal):
    q, k, v, _, qo, ko = make(lq, lk or lq, 12, 4, lead, tail)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal)
    _lib.check_device()
    check_fwd(q, k, v, qo, ko, causal, o, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk,h,hk,causal", CASES)
def test_forward_with_many_heads(lq, lk, h, hk, causal):
    """More than three items per SM, so with a plan (the cases above have one only where they are long)."""
    more = 445 // (h * (sum(lq) // 256 + len(lq) + 2)) + 1
    q, k, v, _, qo, ko = make(lq, lk or lq, h * more, hk * more, 3, 150)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal)
    _lib.check_device()
    check_fwd(q, k, v, qo, ko, causal, o, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [29, 30, 31, 62, 63, 125, 126, 127, 128])
def test_sequences_around_the_warp(n):
    """Without a plan the segments are looked through 32 at a time, up to 126 sequences."""
    lens = [(i * 5) % 3 for i in range(n - 1)] + [4]
    q, k, v, _, qo, ko = make(lens, lens, 1, 1, 1, 2)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, ko, causal=True)
    _lib.check_device()
    check_fwd(q, k, v, qo, ko, True, o, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_large_scores(causal):
    """N(0, 3^2) q and k: row maxima that keep moving, so O is rescaled."""
    q, k, v, _, qo, ko = make([700, 90], [700, 90], 4, 2, std=3.0, seed=1)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal)
    _lib.check_device()
    check_fwd(q, k, v, qo, ko, causal, o, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("n", [1500, 2500])
def test_many_sequences(n, causal):
    """More items than CTAs, more sequences than the plan's threads, one and two tiles in turn; the plan's
    scans in shared memory and in the workspace."""
    lens = [(i * 53) % (301 if n < 2000 else 41) for i in range(n)]
    q, k, v, _, qo, ko = make(lens, lens, 2, 1, seed=2)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, causal=causal)  # k_offsets defaults to q_offsets
    _lib.check_device()
    check_fwd(q, k, v, qo, ko, causal, o, lse)


@pytest.mark.gpu
def test_a_sequence_does_not_see_its_neighbours():
    """Non-finite values of one sequence stay in it; -inf keys and NaN values behind a causal row's tile too."""
    q, k, v, _, qo, ko = make([200, 77, 130], [200, 77, 130], 2, 2, seed=3)
    want, want_lse = wan_flash_packed_fwd(q, k, v, qo, ko, causal=True)
    k[200:277], v[200:277], q[200:277] = float("nan"), float("inf"), float("-inf")
    o, lse = wan_flash_packed_fwd(q, k, v, qo, ko, causal=True)
    for rows in (slice(0, 200), slice(277, None)):
        assert torch.equal(o[rows], want[rows]) and torch.equal(lse[:, rows], want_lse[:, rows])
    assert o[200:277].isnan().all() and lse[:, 200:277].isnan().all()


SPLIT = [
    # few query rows, many keys: walks are cut into pieces
    ([5], [5000], 2, 1, True),
    ([5], [5000], 2, 1, False),
    ([300], [9000], 1, 1, True),                  # two tiles of a record, pieces before and on its diagonal
    ([129, 0, 1, 40], [3000, 700, 4097, 0], 4, 2, True),
    ([129, 0, 1, 40], [3000, 700, 4097, 0], 4, 2, False),
    ([2500], [2500], 2, 2, True),
    ([200, 60], [1800, 20], 3, 3, True),          # 14 blocks: not cut yet
    ([200, 60], [4800, 20], 3, 3, True),          # rows that see nothing beside a cut walk
    ([6000, 1], [6000, 5], 6, 2, True),           # only the longest walks are cut
]


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk,h,hk,causal", SPLIT)
@pytest.mark.parametrize("std", [1.0, 3.0])
def test_cut_walks(lq, lk, h, hk, causal, std):
    q, k, v, _, qo, ko = make(lq, lk, h, hk, 0, 7, std=std, seed=13)
    o, lse, res = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal, residual=True)
    _lib.check_device()
    check_fwd(q, k, v, qo, ko, causal, o, lse)
    # the residual is what one more rounding of the same value takes away
    assert (res.double().abs() <= 2.0**-8 * o.double().abs()).all()
    again, lse2 = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal)
    assert torch.equal(o, again) and torch.equal(lse, lse2)


@pytest.mark.gpu
def test_matches_the_dense_forward_on_one_sequence():
    """One full sequence is wan_flash_fwd's problem: same rounding points, so the same to fp32 sums' order."""
    from wan_flash.interface import wan_flash_fwd

    q, k, v, _, qo, ko = make([640], [640], 2, 2, seed=4)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, ko)
    do, dlse = wan_flash_fwd(q[None], k[None], v[None])
    r = attn64(q, k, v)
    assert_close(do[0], r["o"], r["o_tol"], "dense o")
    assert_close(o, r["o"], r["o_tol"], "packed o")
    assert (lse - dlse[0]).abs().max().item() <= 2 * r["lse_tol"].max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [[0, 60, 50, 100], [-1, 50, 60, 100], [0, 50, 60, 101]])
@pytest.mark.parametrize("which", ["q", "k"])
def test_impossible_offsets(bad, which):
    q, k, v, _, qo, ko = make([50, 10, 40], [50, 10, 40], 2, 1)
    t = torch.tensor(bad, dtype=torch.int32, device="cuda")
    o, lse = wan_flash_packed_fwd(q, k, v, t if which == "q" else qo, t if which == "k" else ko, causal=True)
    with pytest.raises(_lib.WanFlashError):
        _lib.check_device()
    assert o.isnan().all() and lse.isnan().all()
    _lib.check_device()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [[0, 60, 50, 100], [-1, 50, 60, 100], [0, 50, 60, 101]])
def test_impossible_offsets_of_many_heads(bad):
    q, k, v, _, qo, ko = make([50, 10, 40], [50, 10, 40], 100, 50)  # with a plan
    t = torch.tensor(bad, dtype=torch.int32, device="cuda")
    for offs in ((t, ko), (qo, t)):
        o, lse = wan_flash_packed_fwd(q, k, v, *offs, causal=True)
        with pytest.raises(_lib.WanFlashError):
            _lib.check_device()
        assert o.isnan().all() and lse.isnan().all()
        _lib.check_device()


@pytest.mark.gpu
def test_strided_inputs_other_stream_and_replay_with_other_offsets():
    g = torch.Generator().manual_seed(6)
    qkv = torch.randn(400, 3, 2, 128, generator=g).to("cuda", torch.bfloat16)
    qo = offsets([100, 0, 300])
    want = wan_flash_packed_fwd(*(qkv[:, i].contiguous() for i in range(3)), qo, causal=True)
    got = wan_flash_packed_fwd(*(qkv[:, i] for i in range(3)), qo, causal=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q, k, v = (qkv[:, i].contiguous() for i in range(3))
    graphs, outs = [], []
    for _ in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            wan_flash_packed_fwd(q, k, v, qo, causal=True)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(wan_flash_packed_fwd(q, k, v, qo, causal=True))
        graphs.append((graph, side))
    for _ in range(3):
        for graph, side in graphs:
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    for o, lse in outs:
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    qo.copy_(torch.tensor([0, 7, 390, 390], dtype=torch.int32))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    _lib.check_device()
    check_fwd(q, k, v, qo, qo, True, *outs[0])


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_behind_a_kernel_of_another_stream(captured):
    """The first kernel may come up early behind its own stream's last one, never before the stream it waits for."""
    q, k, v, _, qo, ko = make([300, 77], [300, 77], 3, 1)

    def call(x):
        return wan_flash_packed_fwd(x, k, v, qo, ko, causal=True)

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
def test_from_a_thread_without_a_cuda_call_behind_it():
    import threading

    from wan_flash.interface import wan_flash_fwd

    q, k, v, _, qo, ko = make([100], [100], 2, 2)
    want, got = wan_flash_packed_fwd(q, k, v, qo, ko), []
    q4, k4, v4 = q[None], k[None], v[None]
    dense = wan_flash_fwd(q4, k4, v4)
    torch.cuda.synchronize()
    for fn in (lambda: wan_flash_packed_fwd(q, k, v, qo, ko), lambda: wan_flash_fwd(q4, k4, v4)):
        t = threading.Thread(target=lambda: got.append(fn()))
        t.start()
        t.join()
    assert len(got) == 2 and torch.equal(got[0][0], want[0]) and torch.equal(got[1][0], dense[0])


@pytest.mark.gpu
def test_nothing_to_do():
    q, k, v, _, qo, ko = make([0], [5], 2, 1)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, ko)
    assert o.shape == (0, 2, 128) and lse.shape == (2, 0)
    # no sequence at all, and no keys at all
    q, k, v, _, qo, ko = make([30], [0], 2, 1)
    for a, b in ((qo, ko), (qo[:1], ko[:1])):
        o, lse = wan_flash_packed_fwd(q, k, v, a, b, causal=True)
        _lib.check_device()
        assert (o == 0).all() and (lse == float("-inf")).all()


def test_refusals():
    q, k, v, do, qo, ko = make([5, 3], [5, 3], 4, 2, device="cpu")
    for bad in (
        (q, k, v, qo),                          # CPU tensors
        (q.float(), k, v, qo),
        (q[..., :64], k[..., :64], v[..., :64], qo),
        (q[:, :3], k, v, qo),                   # 3 heads over 2
        (q, k, v[:4], qo),
        (q[None], k, v, qo),
        (q, k, v, qo.long()),
        (q, k, v, qo, ko[:2]),
        (q, k, v, qo[:0]),
        (q, k, v, qo[None]),
    ):
        with pytest.raises(AssertionError):
            wan_flash_packed_fwd(*bad)


def test_c_entry_refusals():
    lib = _lib.lib()

    def call(q=16, n=2, tq=8, tk=8, h=4, hk=2, causal=0, ws=1 << 20):
        p = ctypes.c_void_p
        return lib.wf_packed_fwd(p(q) if q else None, *[p(16)] * 8, ws, n, tq, tk, h, hk,
                                 causal, None)

    assert call(n=-1) == -1 and call(h=3) == -1 and call(hk=0) == -1 and call(causal=2) == -1 and call(q=None) == -1
    assert call(q=24) == -3 and call(tq=2**30 + 1) == -2 and call(n=2**25) == -2
    assert call(tq=0) == 0 and call(h=0, hk=0) == 0
    assert lib.wf_packed_fwd_workspace(-1, 1000, 1000, 4, ctypes.byref(ctypes.c_size_t())) == -1


@pytest.mark.gpu
def test_c_entry_refuses_a_small_workspace():
    lib, size, p = _lib.lib(), ctypes.c_size_t(), ctypes.c_void_p
    for tq in (8, 100000):
        assert lib.wf_packed_fwd_workspace(2, tq, 5000, 4, ctypes.byref(size)) == 0
        assert lib.wf_packed_fwd(*[p(16)] * 9, size.value - 1, 2, tq, 5000, 4, 2, 0, None) == -1


@pytest.mark.parametrize("op", [False, True])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_a_forward_mode_tangent_is_refused(monkeypatch, op, which):
    """As wan_flash_attn refuses it, and not dropped: a missing tangent counts as a zero derivative."""
    from torch.autograd import forward_ad

    import wan_flash.packed
    import wan_flash.torch_op

    def launch(q, k, v, q_offsets, k_offsets=None, causal=False, residual=False):
        lse = torch.zeros(q.shape[1], q.shape[0])
        return (torch.zeros_like(q), lse, torch.zeros_like(q)) if residual else (torch.zeros_like(q), lse)

    for module in (wan_flash.packed, wan_flash.torch_op):
        monkeypatch.setattr(module, "wan_flash_packed_fwd", launch)
    fn = wan_flash.torch_op.wan_attention_packed if op else wan_flash.packed.wan_flash_attn_packed
    q, k, v, do, qo, ko = make([5, 3], [5, 3], 4, 2, device="cpu")
    for grad_mode in (False, True):
        with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
            x = [q, k, v]
            x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
            with pytest.raises(NotImplementedError):
                fn(*x, qo, ko)
    assert fn(q, k, v, qo, ko).shape == q.shape


@pytest.mark.parametrize("op", [False, True])
def test_a_forward_mode_tangent_of_the_gradient_is_refused(monkeypatch, op):
    from torch.autograd import forward_ad

    import wan_flash.packed
    import wan_flash.torch_op

    for module in (wan_flash.packed, wan_flash.torch_op):
        monkeypatch.setattr(module, "wan_flash_packed_fwd",
                            lambda q, *a, **kw: (torch.zeros_like(q), torch.zeros(4, 8), torch.zeros_like(q)))
        monkeypatch.setattr(module, "wan_flash_packed_bwd",
                            lambda q, k, v, *a: (torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)))
    q, k, v, do, qo, ko = make([5, 3], [5, 3], 4, 2, device="cpu")
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    o = (wan_flash.torch_op.wan_attention_packed if op else wan_flash.packed.wan_flash_attn_packed)(*leaves, qo, ko)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        torch.autograd.grad(o, leaves, forward_ad.make_dual(do, torch.ones_like(do)), retain_graph=True)
    assert len(torch.autograd.grad(o, leaves, do)) == 3


@pytest.mark.gpu
def test_one_long_sequence_keeps_its_plan_where_its_walks_can_be_cut():
    """1537 to 2048 keys: one sequence with few tiles goes by the plan (a workspace), others without."""
    def planned(n, total, h):
        size = ctypes.c_size_t()
        _lib.check(_lib.lib().wf_packed_fwd_workspace(n, total, total, h, ctypes.byref(size)))
        return size.value > 0

    assert planned(1, 1992, 5) and planned(1, 2048, 1) and planned(1, 1954, 9)
    assert not planned(1, 1992, 15) and not planned(3, 1992, 5) and not planned(1, 1536, 5)
    assert planned(1, 2049, 15)
