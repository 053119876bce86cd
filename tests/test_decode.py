"""Paged decode attention against attention in 64 bits: lengths from nothing to
several CTAs' runs, page sizes that end inside a tile, grouped heads, strided
caches, impossible lengths and pages, graphs, and refusals."""

import ctypes

import pytest
import torch

from tests.attn64 import assert_close, attn64
from wan_flash import _lib
from wan_flash.decode import wan_flash_decode


def make(lens, h, hk, page, seed=0, extra_width=0):
    g = torch.Generator().manual_seed(seed)
    per = [-(-n // page) for n in lens]
    n_pages = sum(per) + 2
    q = torch.randn(len(lens), h, 128, generator=g).to("cuda", torch.bfloat16)
    k = torch.randn(n_pages, page, hk, 128, generator=g).to("cuda", torch.bfloat16)
    v = torch.randn(n_pages, page, hk, 128, generator=g).to("cuda", torch.bfloat16)
    order = torch.randperm(n_pages, generator=g).tolist()
    # entries past a sequence's last page are not read: they point nowhere
    table = torch.full((len(lens), max(per + [0]) + extra_width), 2**31 - 1, dtype=torch.int32)
    for i, n in enumerate(per):
        for j in range(n):
            table[i, j] = order.pop()
    return q, k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def check(q, k, v, table, lengths, o, lse):
    page = k.shape[1]
    for i, n in enumerate(lengths.tolist()):
        at = torch.arange(n, device="cuda")
        pg = table[i].long()[at // page] if n else at
        r = attn64(q[i:i + 1], k[pg, at % page], v[pg, at % page])
        assert_close(o[i:i + 1], r["o"], r["o_tol"], f"o[{i}] of {n}")
        assert_close(lse[i][:, None], r["lse"], r["lse_tol"], f"lse[{i}] of {n}")


def test_refusals():
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    c = torch.zeros(3, 8, 2, 128, dtype=torch.bfloat16)
    t, n = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for bad in (
        (q, c, c, t, n),                        # CPU tensors
        (q.float(), c, c, t, n),
        (q[..., :64], c, c, t, n),
        (q[:, :3], c, c, t, n),                 # 3 heads over 2
        (q, c, c[:2], t, n),
        (q, c, c, t[:1], n),
        (q, c, c, t.long(), n),
        (q, c, c, t, n.long()),
        (q, c, c, t, n[:1]),
        (q, c[:, :0], c[:, :0], t, n),
        (q, c.transpose(2, 3).contiguous().transpose(2, 3), c, t, n),  # rows not contiguous
    ):
        with pytest.raises(AssertionError):
            wan_flash_decode(*bad)


def test_c_entry_refusals():
    lib = _lib.lib()

    def call(q=16, h=4, hk=2, b=1, ws=1 << 30, **kw):
        cfg = _lib.DecodeCfg(3, 8, 3, 0, 3, 2048, 256, 128, 2048, 256, 128)
        for key, x in kw.items():
            setattr(cfg, key, x)
        p = ctypes.c_void_p
        return lib.wf_decode(p(q) if q else None, p(16), p(16), p(16), p(16), p(16), p(16), p(16), ws, b, h, hk,
                             ctypes.byref(cfg), None)

    assert call(b=-1) == -1 and call(h=3) == -1 and call(page_size=0) == -1 and call(q=None) == -1
    assert call(q=24) == -3 and call(k_slot_stride=130) == -3 and call(max_pages=2**30, page_size=2) == -2
    assert call(v_head_stride=-8) == -2 and call(k_page_stride=2**36) == -2
    assert call(n_pages=2**20, k_page_stride=2**16) == -2  # 128 GiB
    assert call(b=0) == 0
    assert lib.wf_decode_workspace(1, 4, 3, 8, 16, ctypes.byref(ctypes.c_size_t())) == -1
    assert lib.wf_decode_workspace(1, 4, 2, 8, 0, ctypes.byref(ctypes.c_size_t())) == -1


@pytest.mark.gpu
def test_c_entry_refuses_a_small_workspace():
    lib, size, p = _lib.lib(), ctypes.c_size_t(), ctypes.c_void_p
    for pages, more in ((32, 0), (33, 1)):  # 512 and 528 tokens of table
        assert lib.wf_decode_workspace(1, 4, 2, pages, 16, ctypes.byref(size)) == 0 and (size.value > 0) == bool(more)
    cfg = _lib.DecodeCfg(3, 16, 33, 0, 33, 4096, 256, 128, 4096, 256, 128)
    for ws, n in ((16, size.value - 1), (None, 0)):
        assert lib.wf_decode(*[p(16)] * 7, p(ws), n, 1, 4, 2, ctypes.byref(cfg), None) == -1


CASES = [
    # lengths, h, h_kv, page size
    ([1], 1, 1, 1),
    ([0], 2, 1, 16),
    ([63, 64, 65, 0, 1], 4, 4, 16),
    ([300], 12, 12, 7),
    ([17, 1000, 129, 0, 4095], 10, 2, 100),
    ([2000, 3], 8, 1, 64),
    ([700, 15], 16, 1, 128),
    ([513, 40], 24, 1, 32),
    ([513, 40], 32, 1, 256),
    ([260, 1], 40, 1, 3),       # two blocks of 20 heads
    ([5000], 3, 3, 1),
    ([20000, 100], 5, 1, 500),  # one row over many CTAs
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,h,hk,page", CASES)
def test_against_64_bits(lens, h, hk, page):
    x = make(lens, h, hk, page, extra_width=1)
    o, lse = wan_flash_decode(*x)
    _lib.check_device()
    assert o.dtype == torch.bfloat16 and lse.dtype == torch.float32
    check(*x, o, lse)
    again, lse2 = wan_flash_decode(*x)
    assert torch.equal(o, again) and torch.equal(lse, lse2)  # the split has a fixed order


@pytest.mark.gpu
@pytest.mark.parametrize("h,hk", [(4, 2), (32, 1), (80, 2)])
@pytest.mark.parametrize("width", [256, 257, 512, 513])
def test_short_tables(h, hk, width):
    """Around the widths up to which a row is one CTA's."""
    for lens in ([width, 0, 1, 200], [64, 65]):
        q, k, v, table, lengths = make(lens, h, hk, 1)
        if table.shape[1] < width:
            table = torch.nn.functional.pad(table, (0, width - table.shape[1]))
        o, lse = wan_flash_decode(q, k, v, table, lengths)
        _lib.check_device()
        check(q, k, v, table, lengths, o, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("h,hk", [(12, 12), (24, 8)])
@pytest.mark.parametrize("longest", [1024, 1025])
def test_more_rows_than_sms(h, hk, longest):
    lens = [(i * 131) % 1000 for i in range(24)] + [longest]
    x = make(lens, h, hk, 1)
    o, lse = wan_flash_decode(*x)
    _lib.check_device()
    check(*x, o, lse)


@pytest.mark.gpu
def test_many_short_sequences():
    lens = [(i * 37) % 90 for i in range(700)]
    x = make(lens, 2, 1, 16)
    o, lse = wan_flash_decode(*x)
    _lib.check_device()
    check(*x, o, lse)


@pytest.mark.gpu
def test_large_scores_and_garbage_behind_the_end():
    """Scores of hundreds (the running maximum moves) and NaN / infinities in every slot that is not in use."""
    q, k, v, table, lengths = make([130, 77, 1], 6, 2, 16)
    q *= 8
    k *= 8
    used = torch.zeros(k.shape[:2], dtype=torch.bool, device="cuda")
    for i, n in enumerate(lengths.tolist()):
        at = torch.arange(n, device="cuda")
        used[table[i].long()[at // 16], at % 16] = True
    k[~used], v[~used] = float("nan"), float("inf")
    o, lse = wan_flash_decode(q, k, v, table, lengths)
    _lib.check_device()
    check(q, k, v, table, lengths, o, lse)


@pytest.mark.gpu
def test_strided_cache_and_queries():
    q, k, v, table, lengths = make([100, 5], 4, 2, 8)
    want = wan_flash_decode(q, k, v, table, lengths)
    both = torch.stack((k, v), 1)                                   # (pages, 2, page, h_kv, 128)
    heads_first = k.transpose(1, 2).contiguous().transpose(1, 2)    # (pages, h_kv, page, 128) in memory
    wide = torch.zeros(2, 4, 256, device="cuda", dtype=torch.bfloat16)
    wide[..., :128] = q
    for args in ((q, both[:, 0], both[:, 1]), (q, heads_first, v), (wide[..., :128], k, v)):
        got = wan_flash_decode(*args, table, lengths)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    tall = torch.zeros(2, 2 * table.shape[1], device="cuda", dtype=torch.int32)
    tall[:, ::2] = table
    got = wan_flash_decode(q, k, v, tall[:, ::2], lengths)
    assert torch.equal(got[0], want[0])


@pytest.mark.gpu
def test_shared_pages():
    """Sequences that share a prefix's pages, and one page in two places of a sequence."""
    q, k, v, table, lengths = make([100, 90, 33], 4, 2, 16)
    table[1, :3] = table[0, :3]
    table[2, 1] = table[2, 0]
    o, lse = wan_flash_decode(q, k, v, table, lengths)
    _lib.check_device()
    check(q, k, v, table, lengths, o, lse)


@pytest.mark.gpu
def test_cache_places_past_32_bits():
    """Pages behind the first 2^31 elements (2^32 bytes) of a cache, by number and by stride."""
    q, k, v, table, lengths = make([300, 17], 4, 2, 16)
    want = wan_flash_decode(q, k, v, table, lengths)
    n, page = k.shape[0], 16 * 2 * 128
    far = 2**31 // page * 9 // 8
    big = torch.empty(2, far + n, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
    big[0, far:], big[1, far:] = k, v
    used = torch.where(table < n, table + far, table)
    spread = torch.as_strided(big, (2, n, 16, 2, 128), (big.stride(0), (far + n) * page // n // 8 * 8, 256, 128, 1))
    for args in ((big[0], big[1], used), (spread[0], spread[1], table)):
        if args[2] is table:
            spread[0], spread[1] = k, v
        got = wan_flash_decode(q, *args, lengths)
        _lib.check_device()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["page", "negative page", "length", "negative length"])
def test_impossible_pages_and_lengths(what):
    q, k, v, table, lengths = make([100, 50, 33], 4, 2, 16)
    if what == "page":
        table[1, 2] = k.shape[0]
    elif what == "negative page":
        table[1, 0] = -5
    elif what == "length":
        lengths[1] = table.shape[1] * 16 + 1
    else:
        lengths[1] = -1
    o, lse = wan_flash_decode(q, k, v, table, lengths)
    with pytest.raises(_lib.WanFlashError):
        _lib.check_device()
    assert o[1].isnan().all() and lse[1].isnan().all()
    rest = [0, 2]  # the others are not touched by it
    check(q[rest], k, v, table[rest], lengths[rest], o[rest], lse[rest])
    _lib.check_device()


@pytest.mark.gpu
def test_impossible_pages_and_lengths_of_long_rows():
    """As above where rows are split over CTAs: sequences 1 (a page) and 3 (the length) are lost, no other."""
    q, k, v, table, lengths = make([900, 1500, 33, 700], 4, 2, 16)
    table[1, 60] = k.shape[0]
    lengths[3] = table.shape[1] * 16 + 1
    o, lse = wan_flash_decode(q, k, v, table, lengths)
    with pytest.raises(_lib.WanFlashError):
        _lib.check_device()
    assert o[[1, 3]].isnan().all() and lse[[1, 3]].isnan().all()
    rest = [0, 2]
    check(q[rest], k, v, table[rest], lengths[rest], o[rest], lse[rest])
    _lib.check_device()


@pytest.mark.gpu
@pytest.mark.parametrize("long", [300, 3000])  # whole rows, and rows over several CTAs
def test_captured_graphs_side_by_side_with_changing_lengths(long):
    xs = [make([90, long], 4, 2, 16, seed=s) for s in range(2)]
    want = [wan_flash_decode(*x) for x in xs]
    graphs, outs = [], []
    for x in xs:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            wan_flash_decode(*x)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(wan_flash_decode(*x))
        graphs.append((graph, side))
    for _ in range(5):  # both at once: workspaces of their own
        for graph, side in graphs:
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    for (o, lse), (wo, wl) in zip(outs, want):
        assert torch.equal(o, wo) and torch.equal(lse, wl)
    xs[0][4].copy_(torch.tensor([1, long - 1], dtype=torch.int32))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    _lib.check_device()
    check(*xs[0], *outs[0])


@pytest.mark.gpu
def test_nothing_to_do():
    q, k, v, table, lengths = make([4], 4, 2, 16)
    o, lse = wan_flash_decode(q[:0], k, v, table[:0], lengths[:0])
    assert o.shape == (0, 4, 128) and lse.shape == (0, 4)
    # an empty cache with empty sequences
    o, lse = wan_flash_decode(q, k[:0], v[:0], table[:, :0], lengths * 0)
    _lib.check_device()
    assert (o == 0).all() and (lse == float("-inf")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_behind_a_kernel_of_another_stream(captured):
    """The first kernel may come up early behind its own stream's last one, never before the stream it waits for."""
    q, k, v, table, lengths = make([300, 17, 1000], 4, 2, 16)

    def call(x):
        return wan_flash_decode(x, k, v, table, lengths)

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
@pytest.mark.parametrize("h,hk", [(6, 2), (12, 1), (20, 1), (32, 1)])  # one to four blocks of 8 heads a row
@pytest.mark.parametrize("extra_width", [0, 300])  # a CTA per row, and runs of tiles with a join
def test_probabilities_are_not_rounded_to_bf16(h, hk, extra_width):
    """o is off by its own rounding and by fp32 errors only.

    q is 0 but in its first dim, so a score is one exact product.  What is left, relative to a
    probability: its exponent (three roundings of at most 2 in log2 units, ln 2 * 3 * 2 * 2^-24)
    and exp2 (2^-22), together below 2^-20, and 2^-16 from the pair of bf16 that it is multiplied as.  An
    output adds 16 products of either half a step of 64 tokens, then 4 warps and a few CTAs' runs:
    an fp32 step of the row's sum of |p v| each at most.  The sum of the row, 300 fp32 additions, is
    below 2^-15 of o.  A probability rounded to one bf16 would be 2^-8 off."""
    from tests.attn64 import E32, U

    lens = [300, 40, 130, 17]
    q, k, v, table, lengths = make(lens, h, hk, 16, seed=21, extra_width=extra_width)
    q[..., 1:] = 0
    q.clamp_(-2, 2)
    o, lse = wan_flash_decode(q, k, v, table, lengths)
    _lib.check_device()
    check(q, k, v, table, lengths, o, lse)
    for i, n in enumerate(lens):
        at = torch.arange(n, device="cuda")
        pg = table[i].long()[at // 16]
        r = attn64(q[i:i + 1], k[pg, at % 16], v[pg, at % 16])
        spread = (r["p"] @ v[pg, at % 16].double().transpose(0, 1).repeat_interleave(h // hk, 0).abs()).transpose(0, 1)
        fp32 = (2.0**-16 + 2.0**-20 + (2 * 16 * -(-n // 64) + 16) * E32) * spread + 2.0**-15 * r["o"].abs()
        assert_close(o[i:i + 1], r["o"], fp32 + U * (r["o"].abs() + fp32), f"o[{i}] of {n}")


@pytest.mark.gpu
@pytest.mark.parametrize("h,hk", [(6, 2), (32, 1)])
@pytest.mark.parametrize("extra_width", [0, 300])
def test_infinite_values_stay_infinite(h, hk, extra_width):
    """A visible token whose value is infinite in a dim makes o infinite there (every probability is above 0), with its
    sign; two of opposite signs, or a NaN, make NaN; the other dims are as without."""
    lens = [300, 1, 17, 130]
    q, k, v, table, lengths = make(lens, h, hk, 16, seed=22, extra_width=extra_width)
    want, want_lse = wan_flash_decode(q, k, v, table, lengths)
    inf = float("inf")
    for i, n in enumerate(lens):
        for dim, at, x in ((3, 0, inf), (4, n - 1, -inf), (5, n // 2, inf), (6, 0, inf), (6, n - 1, -inf), (127, n // 3, float("nan"))):
            v[table[i, at // 16].long(), at % 16, :, dim] = x
    o, lse = wan_flash_decode(q, k, v, table, lengths)
    _lib.check_device()
    assert torch.equal(lse, want_lse)
    for i, n in enumerate(lens):
        assert (o[i, :, 3] == inf).all() and (o[i, :, 4] == -inf).all() and (o[i, :, 5] == inf).all()
        assert (o[i, :, 6].isnan() if n > 1 else o[i, :, 6] == -inf).all() and o[i, :, 127].isnan().all()
        rest = [d for d in range(128) if d not in (3, 4, 5, 6, 127)]
        assert torch.equal(o[i][:, rest], want[i][:, rest])
