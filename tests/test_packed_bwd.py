"""Packed attention, backward: gradients against the formulas in 64 bits and
against differences, the splits and the ordered mode, NaN outside the
sequences, graphs, and refusals."""

import pytest
import torch

from tests.attn64 import U, assert_close, attn64, grads64
from tests.test_packed import CASES, make, offsets
from wan_flash import _lib, features
from wan_flash.packed import wan_flash_attn_packed, wan_flash_packed_bwd, wan_flash_packed_fwd


@pytest.fixture(autouse=True)
def _reset_features():
    yield
    features.reset()


def check_bwd(q, k, v, do, qo, ko, causal, dq, dk, dv, residual=False):
    qo, ko = qo.tolist(), ko.tolist()
    for i in range(len(qo) - 1):
        a, b, c, d = qo[i], qo[i + 1], ko[i], ko[i + 1]
        if a == b or c == d:
            assert (dq[a:b] == 0).all() and (dk[c:d] == 0).all() and (dv[c:d] == 0).all()
            continue
        want = grads64(q[a:b], k[c:d], v[c:d], do[a:b], causal, residual)
        for name, got in (("dq", dq[a:b]), ("dk", dk[c:d]), ("dv", dv[c:d])):
            assert_close(got, *want[name], f"{name} of sequence {i}")
    for x, off in ((dq, qo), (dk, ko), (dv, ko)):
        assert (x[:off[0]] == 0).all() and (x[off[-1]:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk,h,hk,causal", CASES)
@pytest.mark.parametrize("lead,tail", [(0, 0), (3, 150)])
def test_backward(lq, lk, h, hk, causal, lead, tail):
    q, k, v, do, qo, ko = make(lq, lk or lq, h, hk, lead, tail)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal)
    grads = wan_flash_packed_bwd(q, k, v, o, lse, do, qo, ko, causal=causal)
    _lib.check_device()
    assert all(g.shape == x.shape and g.dtype == x.dtype for g, x in zip(grads, (q, k, v)))
    check_bwd(q, k, v, do, qo, ko, causal, *grads)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nsplit,deterministic", [(1, True), (2, False), (3, True), (7, False), (40, True)])
def test_splits_and_ordered_mode(nsplit, deterministic, causal):
    lq, lk = [700, 1, 129, 0], [700, 40, 300, 5]
    q, k, v, do, qo, ko = make(lq, lk, 6, 2, 1, 9, seed=7)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal)
    features.set_bwd_overrides(nsplit=nsplit, deterministic=deterministic)
    grads = wan_flash_packed_bwd(q, k, v, o, lse, do, qo, ko, causal=causal)
    _lib.check_device()
    check_bwd(q, k, v, do, qo, ko, causal, *grads)
    for _ in range(2):
        again = wan_flash_packed_bwd(q, k, v, o, lse, do, qo, ko, causal=causal)
        assert torch.equal(grads[1], again[1]) and torch.equal(grads[2], again[2])
        if deterministic:
            assert torch.equal(grads[0], again[0])


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("n", [1200, 2500])  # the plan's scans in shared memory, and in the workspace
def test_many_sequences(n, causal):
    lens = [(i * 53) % (301 if n < 2000 else 41) for i in range(n)]
    q, k, v, do, qo, ko = make(lens, lens, 2, 1, seed=2)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, causal=causal)
    grads = wan_flash_packed_bwd(q, k, v, o, lse, do, qo, causal=causal)
    _lib.check_device()
    check_bwd(q, k, v, do, qo, ko, causal, *grads)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_large_scores(causal):
    q, k, v, do, qo, ko = make([400, 90], [400, 90], 4, 2, std=3.0, seed=1)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal)
    grads = wan_flash_packed_bwd(q, k, v, o, lse, do, qo, ko, causal=causal)
    _lib.check_device()
    check_bwd(q, k, v, do, qo, ko, causal, *grads)


@pytest.mark.gpu
def test_a_sequence_does_not_see_its_neighbours():
    features.set_bwd_overrides(deterministic=True)
    q, k, v, do, qo, ko = make([200, 77, 130], [200, 77, 130], 2, 2, seed=3)

    def grads():
        o, lse = wan_flash_packed_fwd(q, k, v, qo, ko, causal=True)
        return wan_flash_packed_bwd(q, k, v, o, lse, do, qo, ko, causal=True)

    want = grads()
    for x in (q, k, v, do):
        x[200:277] = float("nan")
    for g, w in zip(grads(), want):
        assert torch.equal(g[:200], w[:200]) and torch.equal(g[277:], w[277:])
        assert g[200:277].isnan().any()


@pytest.mark.gpu
def test_rows_that_see_no_key_reach_no_gradient():
    features.set_bwd_overrides(deterministic=True)
    lq, lk = [200, 300, 141], [130, 5, 140]
    q, k, v, do, qo, ko = make(lq, lk, 4, 2, seed=6)

    def grads():
        o, lse, res = wan_flash_packed_fwd(q, k, v, qo, ko, causal=True, residual=True)
        return o, *wan_flash_packed_bwd(q, k, v, o, lse, do, qo, ko, causal=True, o_residual=res)

    want = grads()
    for a, n, m in zip(qo.tolist(), lq, lk):  # the first n - m rows of each
        assert (want[0][a:a + n - m] == 0).all() and (want[1][a:a + n - m] == 0).all()
        q[a:a + n - m] = float("nan")
        do[a:a + n - m] = float("nan")
    for g, w in zip(grads(), want):
        assert torch.equal(g, w)


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk,h,hk,causal", CASES)
def test_residual_of_o(lq, lk, h, hk, causal):
    """o + residual is o to 16 bits, and with it dq and dk do not carry o's rounding through D."""
    q, k, v, do, qo, ko = make(lq, lk or lq, h, hk, 2, 130)
    o, lse, res = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal, residual=True)
    plain, plain_lse = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal)
    assert torch.equal(o, plain) and torch.equal(lse, plain_lse)
    grads = wan_flash_packed_bwd(q, k, v, o, lse, do, qo, ko, causal=causal, o_residual=res)
    _lib.check_device()
    check_bwd(q, k, v, do, qo, ko, causal, *grads, residual=True)
    qo, ko = qo.tolist(), ko.tolist()
    for i in range(len(qo) - 1):
        a, b, c, d = qo[i], qo[i + 1], ko[i], ko[i + 1]
        if a < b:
            r = attn64(q[a:b], k[c:d], v[c:d], causal)
            # p's rounding stays; o's own step (2^-8) becomes its square
            tol = r["o_tol"] - U * r["o"].abs() + U * U * (r["o"].abs() + r["o_tol"])
            assert_close(o[a:b].double() + res[a:b].double(), r["o"], tol, f"o + residual of sequence {i}")
    assert (res[:qo[0]] == 0).all() and (res[qo[-1]:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_autograd_and_differences(causal):
    """The gradient along a direction against a central difference of the function in 64 bits."""
    q, k, v, do, qo, ko = make([150, 37], [170, 37], 4, 2, seed=8)
    g = torch.Generator().manual_seed(9)
    move = [torch.randn(x.shape, generator=g).to("cuda").double() for x in (q, k, v)]
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    o = wan_flash_attn_packed(*leaves, qo, ko, causal=causal)
    grads = torch.autograd.grad(o, leaves, do)
    _lib.check_device()

    def loss(step):
        total = 0.0
        for a, b, c, d in ((0, 150, 0, 170), (150, 187, 170, 207)):
            x, y, z = ((t.double() + step * m)[s] for t, m, s in zip((q, k, v), move, (slice(a, b), slice(c, d), slice(c, d))))
            total += (attn64(x, y, z, causal)["o"] * do[a:b].double()).sum().item()
        return total

    h = 1e-5  # the difference itself is off by h^2 / 6 of the third derivative and 1e-16 / h of the loss: below 1e-6
    want = (loss(h) - loss(-h)) / (2 * h)
    got = sum((x.double() * m).sum().item() for x, m in zip(grads, move))
    tol = 0.0
    for a, b, c, d in ((0, 150, 0, 170), (150, 187, 170, 207)):
        w = grads64(q[a:b], k[c:d], v[c:d], do[a:b], causal)
        tol += sum((w[n][1] * m[s].abs()).sum().item()
                   for n, m, s in zip(("dq", "dk", "dv"), move, (slice(a, b), slice(c, d), slice(c, d))))
    assert abs(got - want) <= tol + 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [[0, 60, 50, 100], [-1, 50, 60, 100], [0, 50, 60, 101]])
def test_impossible_offsets(bad):
    q, k, v, do, qo, ko = make([50, 10, 40], [50, 10, 40], 2, 1)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, ko)
    t = torch.tensor(bad, dtype=torch.int32, device="cuda")
    for args in ((t, ko), (qo, t)):
        grads = wan_flash_packed_bwd(q, k, v, o, lse, do, *args)
        with pytest.raises(_lib.WanFlashError):
            _lib.check_device()
        assert all(x.isnan().all() for x in grads)
    _lib.check_device()


@pytest.mark.gpu
def test_one_derivative_only_and_expanded_gradients():
    q, k, v, do, qo, _ = make([100, 40], [100, 40], 2, 1)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    o = wan_flash_attn_packed(*leaves, qo)
    one = torch.ones((), device="cuda", dtype=torch.bfloat16).expand(o.shape)  # as from o.sum()
    grads = torch.autograd.grad(o, leaves, one, retain_graph=True)
    _lib.check_device()
    check_bwd(q, k, v, one, qo, qo, False, *grads, residual=True)
    (dq,) = torch.autograd.grad(o, leaves[0], do, create_graph=True)
    with pytest.raises(RuntimeError):
        dq.sum().backward()


@pytest.mark.gpu
def test_training_step_captured_and_replayed_with_other_offsets():
    q, k, v, do, qo, ko = make([300, 77], [300, 77], 4, 2, seed=11)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        o = wan_flash_attn_packed(*leaves, qo, causal=True)
        return o, *torch.autograd.grad(o, leaves, do)

    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for lens in ([300, 77], [1, 376], [377, 0]):
        qo.copy_(offsets(lens))
        graph.replay()
        torch.cuda.synchronize()
        _lib.check_device()
        check_bwd(q, k, v, do, qo, qo, True, *out[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("deterministic", [False, True])
def test_captured_behind_a_copy(deterministic):
    """A graph whose nodes before the kernels are copies and (in ordered mode) a memset."""
    features.set_bwd_overrides(deterministic=deterministic)
    q, k, v, do, qo, ko = make([300, 77], [300, 77], 4, 2)
    x = torch.zeros_like(q)

    def run():
        x.copy_(q)
        o, lse = wan_flash_packed_fwd(x, k, v, qo, ko, causal=True)
        return wan_flash_packed_bwd(x, k, v, o, lse, do, qo, ko, causal=True)

    want = run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(3):
        x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for name, g, w in zip(("dq", "dk", "dv"), got, want):
            if deterministic or name != "dq":
                assert torch.equal(g, w), name
        check_bwd(q, k, v, do, qo, ko, True, *got)
    _lib.check_device()


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_rows_past_32_bits(causal):
    """Sequences behind 2^31 elements give what they give at the start, bit for bit
    (with whole walks: the number of key tiles, padding's too, decides on pieces)."""
    features.set_bwd_overrides(nsplit=1, deterministic=True)
    h, lens = 16, [300, 1, 140]
    q, k, v, do, qo, ko = make(lens, lens, h, h)
    o, lse, res = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal, residual=True)
    want = o, lse, *wan_flash_packed_bwd(q, k, v, o, lse, do, qo, ko, causal=causal, o_residual=res)
    lead, n = 2**31 // (h * 128) + 77, sum(lens)
    big = []
    for x in (q, k, v, do):
        big.append(torch.empty(lead + n, h, 128, dtype=torch.bfloat16, device="cuda"))
        big[-1][lead:] = x
    at = (qo + lead).int()
    o, lse, res = wan_flash_packed_fwd(*big[:3], at, causal=causal, residual=True)
    got = o, lse, *wan_flash_packed_bwd(*big[:3], o, lse, big[3], at, causal=causal, o_residual=res)
    _lib.check_device()
    for g, w in zip(got, want):
        g, w = (g[:, lead:], w) if g is lse else (g[lead:], w)
        assert torch.equal(g, w)
    assert not o[:lead].any() and not got[2][:lead].any()


@pytest.mark.gpu
@pytest.mark.parametrize("lens,h,hk,causal", [([256] * 40, 8, 8, False), ([4000], 12, 12, False), ([900, 2300, 17], 16, 4, True)])
def test_dk_and_dv_are_reproducible(lens, h, hk, causal):
    q, k, v, do, qo, ko = make(lens, lens, h, hk)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal)
    _, dk, dv = wan_flash_packed_bwd(q, k, v, o, lse, do, qo, ko, causal=causal)
    for _ in range(5):
        again = wan_flash_packed_bwd(q, k, v, o, lse, do, qo, ko, causal=causal)
        assert torch.equal(again[1], dk) and torch.equal(again[2], dv)


@pytest.mark.gpu
def test_c_entry_refuses_a_small_workspace():
    import ctypes

    lib, cfg, size = _lib.lib(), _lib.PackedBwdCfg(0, 0), ctypes.c_size_t()
    assert lib.wf_packed_bwd_workspace(2, 8, 8, 4, 2, ctypes.byref(cfg), ctypes.byref(size)) == 0
    p = ctypes.c_void_p
    assert lib.wf_packed_bwd(*[p(16)] * 13, size.value - 1, 2, 8, 8, 4, 2, 0, ctypes.byref(cfg), None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_long_walks_are_cut_into_pieces(causal):
    """One sequence, one key-value head for 8 q heads: 17 key tiles, cut by the device."""
    q, k, v, do, qo, ko = make([2100], [2100], 8, 1, seed=12)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal)
    grads = wan_flash_packed_bwd(q, k, v, o, lse, do, qo, ko, causal=causal)
    _lib.check_device()
    check_bwd(q, k, v, do, qo, ko, causal, *grads)


@pytest.mark.gpu
def test_no_queries_or_no_keys():
    for lq, lk in (([0], [5]), ([5], [0])):
        q, k, v, do, qo, ko = make(lq, lk, 2, 1)
        leaves = [x.requires_grad_() for x in (q, k, v)]
        o = wan_flash_attn_packed(*leaves, qo, ko)
        for g, x in zip(torch.autograd.grad(o, leaves, do), leaves):
            assert g.shape == x.shape and (g == 0).all()
        _lib.check_device()


def test_refusals():
    q, k, v, do, qo, ko = make([5, 3], [5, 3], 4, 2, device="cpu")
    lse = torch.zeros(4, 8)
    for bad in (
        (q, k, v, q, lse, do, qo),                  # CPU tensors
        (q, k, v, q, lse.double(), do, qo),
        (q, k, v, q, lse[:, :7], do, qo),
        (q, k, v, q[:7], lse, do, qo),
        (q, k, v, q, lse, do.float(), qo),
    ):
        with pytest.raises(AssertionError):
            wan_flash_packed_bwd(*bad)


def test_c_entry_refusals():
    import ctypes

    lib = _lib.lib()
    size = ctypes.c_size_t()
    cfg = _lib.PackedBwdCfg(1, 0)

    def call(n=2, tq=8, tk=8, h=4, hk=2, causal=0, nsplit=1, ws=1 << 30, q=16):
        c = _lib.PackedBwdCfg(nsplit, 0)
        p = ctypes.c_void_p
        return lib.wf_packed_bwd(p(q) if q else None, *[p(16)] * 12, ws, n, tq, tk, h, hk, causal, ctypes.byref(c), None)

    assert call(n=-1) == -1 and call(hk=3) == -1 and call(nsplit=-1) == -1 and call(nsplit=2000) == -1 and call(causal=3) == -1 and call(q=None) == -1
    assert call(q=8) == -3 and call(tq=0) == -2 and call(tk=0) == -2
    assert call(h=0, hk=0) == 0 and call(tq=0, tk=0) == 0
    assert lib.wf_packed_bwd_workspace(2, 8, 8, 4, 3, ctypes.byref(cfg), ctypes.byref(size)) == -1
    assert lib.wf_packed_bwd_workspace(2, 8, 8, 4, 2, None, ctypes.byref(size)) == -1


def _workspace(n, total_q, total_k, h, hk, nsplit=0, deterministic=0):
    import ctypes

    cfg, size = _lib.PackedBwdCfg(nsplit, deterministic), ctypes.c_size_t()
    _lib.check(_lib.lib().wf_packed_bwd_workspace(n, total_q, total_k, h, hk, ctypes.byref(cfg), ctypes.byref(size)))
    return size.value


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,h,hk", [(50000, 2500, 40, 40), (32768, 2048, 32, 8), (1000, 100000, 16, 16)])
def test_workspace_grows_with_rows_not_with_sequences(rows, n, h, hk):
    """512 bytes a row and head of fp32 dq; a head and tile of 128 rows 4 KiB (its rows rounded up to 8) and
    1 KiB of lse and D; less than 1 KiB of records a tile, 64 bytes a sequence; and what one sequence of these
    rows needs for pieces."""
    tiles = min(rows, rows // 128 + n + 2)
    most = _workspace(1, rows, rows, h, hk) + 5 * 1024 * h * tiles + 1024 * tiles + 64 * n
    assert _workspace(n, rows, rows, h, hk) <= most
    assert _workspace(n, rows, rows, h, hk, 1, 1) <= most


@pytest.mark.gpu
def test_workspace_of_a_set_split_is_bounded_by_the_units():
    """A walk over group * query tiles units makes no more pieces than that."""
    assert _workspace(1, 100, 100, 4, 2, 1024) == _workspace(1, 100, 100, 4, 2, 4)
    assert _workspace(3, 100, 3000, 4, 2, 1024) <= _workspace(3, 100, 3000, 4, 2, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nsplit,deterministic", [(0, False), (5, True)])
def test_sequence_ends_at_every_place_of_a_tile(causal, nsplit, deterministic):
    lq = [1, 63, 64, 65, 127, 128, 129, 191, 0, 192, 193, 2, 256, 319, 320, 321, 8, 62]
    lk = [5, 64, 63, 200, 127, 129, 128, 1, 7, 300, 193, 0, 256, 30, 321, 320, 9, 63]
    q, k, v, do, qo, ko = make(lq, lk, 4, 2, 5, 70, seed=13)
    o, lse = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal)
    features.set_bwd_overrides(nsplit=nsplit, deterministic=deterministic)
    grads = wan_flash_packed_bwd(q, k, v, o, lse, do, qo, ko, causal=causal)
    _lib.check_device()
    check_bwd(q, k, v, do, qo, ko, causal, *grads)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,h,hk", [([3000, 200], 6, 2), ([700], 2, 2), ([2500], 1, 1)])  # whole walks, no plan, cut walks
def test_feature_switches(lens, h, hk):
    """rescale_skip_threshold moves the roundings (the row maximum grows by less than 8 log2 units over the
    blocks), num_sms and pdl move none."""
    q, k, v, do, qo, ko = make(lens, lens, h, hk, seed=14)

    def run():
        o, lse, res = wan_flash_packed_fwd(q, k, v, qo, ko, residual=True)
        return o, lse, *wan_flash_packed_bwd(q, k, v, o, lse, do, qo, ko, o_residual=res)

    want = run()
    for a, b in zip(qo.tolist(), qo.tolist()[1:]):
        r = attn64(q[a:b], k[a:b], v[a:b])
        assert_close(want[0][a:b], r["o"], r["o_tol"], "o")
    features.set_bwd_overrides(pdl=False)
    for sms in (0, 1, 7, 500, 2**31 - 1):
        features.set_overrides(num_sms=sms)
        got = run()
        for i in (0, 1, 3, 4):
            assert torch.equal(got[i], want[i])
        check_bwd(q, k, v, do, qo, ko, False, *got[2:], residual=True)
    features.set_overrides(num_sms=0, rescale_skip_threshold=0.0)
    got = run()
    _lib.check_device()
    assert not torch.equal(got[0], want[0])
    for a, b in zip(qo.tolist(), qo.tolist()[1:]):
        r = attn64(q[a:b], k[a:b], v[a:b])
        assert_close(got[0][a:b], r["o"], r["o_tol"], "o")
        assert_close(got[1][:, a:b], r["lse"], r["lse_tol"], "lse")


def test_feature_switches_reach_the_c_call(monkeypatch):
    """What the calls pass on, with a stand-in for the launch."""
    import wan_flash.packed as packed

    calls = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: calls.append((name, a)) or 0

    monkeypatch.setattr(packed._lib, "lib", lambda: Lib())
    monkeypatch.setattr(packed, "_launch", lambda fn, device, *a: fn(*a))
    monkeypatch.setattr(packed, "_check", lambda q, k, v, a, b: (8, 8, 4, 2, 2, q.device))
    monkeypatch.setattr(packed, "_fwd_bytes", lambda *a: 0)
    sizes = {}
    monkeypatch.setattr(packed, "_bwd_cfg_bytes", lambda *a: sizes.setdefault("args", a) and (None, 0))
    q, k, v, do, qo, ko = make([5, 3], [5, 3], 4, 2, device="cpu")
    features.set_overrides(rescale_skip_threshold=0.0, num_sms=3)
    features.set_bwd_overrides(pdl=False, nsplit=2, deterministic=True)
    o, lse = packed.wan_flash_packed_fwd(q, k, v, qo, ko)
    name, args = calls[-1]
    assert name == "wf_packed_fwd_with" and (args[-1].rescale_threshold, args[-1].num_sms) == (0.0, 3)
    packed.wan_flash_packed_bwd(q, k, v, o, lse, do, qo, ko)
    assert calls[-1][0] == "wf_packed_bwd_with" and sizes["args"][-3:] == (2, True, False)


def test_c_entries_with_options_refuse():
    import ctypes

    p, lib = ctypes.c_void_p, _lib.lib()
    bad = _lib.FwdCfg(8.0, 0, -1, 0)
    assert lib.wf_packed_fwd_with(*[p(16)] * 9, 1 << 30, 2, 8, 8, 4, 2, 0, ctypes.byref(bad), None) == -1
    for cfg, want in ((None, -1), (ctypes.byref(_lib.BwdCfg(-1, 1)), -1), (ctypes.byref(_lib.BwdCfg(2000, 1)), -1)):
        assert lib.wf_packed_bwd_with(*[p(16)] * 13, 1 << 30, 2, 8, 8, 4, 2, 0, cfg, None) == want


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk", [([1500, 1100], [1500, 1100]), ([300, 700], [1500, 700]), ([900, 200], [140, 1300])])
@pytest.mark.parametrize("causal", [False, True])
def test_each_gradient_depends_on_the_visible_rows_and_keys_alone(lq, lk, causal):
    """One key of a long row more or less would pass the bounds of the sums; so another key (or row) is put in place
    of one: what does not see it stays bit for bit, and the first row (last key) that does see it changes.  (A
    row that sees one key has p = 1 and dS = p (dP - D) = 0 whatever that key is: no dq, and nothing for dk.)"""
    features.set_bwd_overrides(nsplit=1, deterministic=True)
    q, k, v, do, qo, ko = make(lq, lk, 4, 2, seed=15)

    def run(q, k, v, do):
        o, lse, res = wan_flash_packed_fwd(q, k, v, qo, ko, causal=causal, residual=True)
        return o, *wan_flash_packed_bwd(q, k, v, o, lse, do, qo, ko, causal=causal, o_residual=res)

    def differ(a, b):  # per row, whether all heads differ / any head differs
        d = (a != b).any(-1)
        return d.all(-1), d.any(-1)

    want = run(q, k, v, do)
    a0, c0 = 0, 0
    for a, c in zip(lq, lk):
        for t in (0, 1, 127, 128, c // 2, c - 1):  # key t is seen by rows >= t - (c - a)
            k2, v2 = k.clone(), v.clone()
            k2[c0 + t], v2[c0 + t] = k[c0 + t].flip(-1), v[c0 + t].flip(-1)
            got = run(q, k2, v2, do)
            first = max(0, t - (c - a)) if causal else 0
            for i in (0, 1):  # o, dq
                every, some = differ(got[i], want[i])
                assert not some[:a0 + first].any() and not some[a0 + a:].any()
                alone = causal and first + 1 + c - a == 1
                assert (alone and i == 1) or every[a0 + first]
                assert every[a0 + a - 1]
        for r in (0, 1, 127, 128, a // 2, a - 1):  # row r sees keys < r + 1 + c - a
            q2, do2 = q.clone(), do.clone()
            q2[a0 + r], do2[a0 + r] = q[a0 + r].flip(-1), do[a0 + r].flip(-1)
            got = run(q2, k, v, do2)
            seen = max(0, min(c, r + 1 + c - a)) if causal else c
            for i in (2, 3):  # dk, dv
                every, some = differ(got[i], want[i])
                assert not some[:c0].any() and not some[c0 + seen:].any()
                assert seen == 0 or (seen == 1 and i == 2) or (every[c0] and every[c0 + seen - 1])
        a0, c0 = a0 + a, c0 + c


@pytest.mark.gpu
@pytest.mark.parametrize("deterministic", [False, True])
def test_two_backwards_side_by_side_on_two_streams(deterministic):
    features.set_bwd_overrides(deterministic=deterministic)
    work = []
    for seed, lens in ((16, [900, 33, 1200]), (17, [1500, 640, 1])):
        q, k, v, do, qo, ko = make(lens, lens, 8, 2, seed=seed)
        o, lse, res = wan_flash_packed_fwd(q, k, v, qo, ko, causal=True, residual=True)
        work.append((q, k, v, o, lse, do, qo, ko, True, res))
    want = [wan_flash_packed_bwd(*w) for w in work]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [[], []]
        for _ in range(3):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(wan_flash_packed_bwd(*work[i]))
        torch.cuda.synchronize()
        for i in range(2):
            for g in got[i]:
                assert torch.equal(g[1], want[i][1]) and torch.equal(g[2], want[i][2])
                if deterministic:
                    assert torch.equal(g[0], want[i][0])
                else:  # sums of the same contributions in another order: an fp32 step of each, then a rounding
                    check_bwd(*work[i][:3], work[i][5], work[i][6], work[i][7], True, *g, residual=True)
    _lib.check_device()
