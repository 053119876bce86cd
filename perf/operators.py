"""Cases and plain forms of the operators around packed and cached attention.

Three operators, reached through the package's public entry points:

* ``rope``    rotary positions with three axes (time, height, width) of q and k:
              ``wan_flash.rope.wan_flash_rope(q, k, positions, table)``.
              Pair i of the 128 head dims, (x[2i], x[2i+1]), turns by the angle
              positions[token, axis(i)] * theta^(-2 j / d_axis), j the pair's place in
              its axis; pairs 0-21 belong to time, 22-42 to height, 43-63 to width.
              A token with a negative position is padding and passes unchanged.
* ``packed``  softmax attention over sequences of different lengths packed one behind
              the other, grouped heads, causal or not, forward and backward:
              ``wan_flash.packed.wan_flash_packed_fwd(q, k, v, q_offsets, k_offsets, causal)``
              and ``wan_flash_attn_packed`` (differentiable).  Causal: query i of a
              sequence with lq queries and lk keys sees keys j <= i + lk - lq; a row that
              sees no key gives o = 0 and lse = -inf.
* ``decode``  attention of one new token per sequence over a paged key-value cache:
              ``wan_flash.decode.wan_flash_decode(q, k_cache, v_cache, page_table, lengths)``.

``own`` false: the plain forms (elementary torch operations in fp32, rounded once).
``own`` true: the framework's kernels.
"""

import math

import torch

own = False

D = 128
SCALE = 1.0 / math.sqrt(D)
AXES = (44, 42, 42)  # head dims turned by time, height, width
THETA = 10000.0
MAX_POS = 1024  # rows of the rotary table, as the Wan models keep them


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one denoising/decoding step's new tokens of 8 streams: pure latency
        {"name": "rope_step", "op": "rope", "b": 8, "t": 1, "hh": 1, "ww": 1, "h": 12, "hk": 12, "pad": 0,
         "dtype": "bf16", "train": False},
        # 480p self attention's q and k (21 x 30 x 52 latent tokens, 12 heads), with gradients
        {"name": "rope_480p_train", "op": "rope", "b": 1, "t": 21, "hh": 30, "ww": 52, "h": 12, "hk": 12, "pad": 0,
         "dtype": "bf16", "train": True},
        # 720p self attention's q and k of the 40-head model
        {"name": "rope_720p", "op": "rope", "b": 1, "t": 21, "hh": 45, "ww": 80, "h": 40, "hk": 40, "pad": 0,
         "dtype": "bf16", "train": False},
        # fp32 activations, grouped heads, an odd grid with padding tokens behind it, a batch
        {"name": "rope_fp32_odd", "op": "rope", "b": 3, "t": 7, "hh": 31, "ww": 33, "h": 10, "hk": 2, "pad": 37,
         "dtype": "fp32", "train": False},
        # a few short prompts, among them a single token and an empty one
        {"name": "packed_fwd_short", "op": "packed", "lq": "77,1,0,130,257", "lk": "77,1,0,130,257", "h": 12, "hk": 4,
         "causal": True, "train": False},
        # images (1 x 30 x 52 tokens) and clips (5 and 3 latent frames) packed in one batch, all heads
        {"name": "packed_fwd_clips", "op": "packed", "lq": "1560,7800,1560,4680", "lk": "1560,7800,1560,4680",
         "h": 12, "hk": 12, "causal": False, "train": False},
        # long causal prompts with grouped heads
        {"name": "packed_fwd_causal", "op": "packed", "lq": "16384,1000", "lk": "16384,1000", "h": 16, "hk": 4,
         "causal": True, "train": False},
        # training on ragged causal sequences, grouped heads
        {"name": "packed_train_causal", "op": "packed", "lq": "4097,333,2048,1,900", "lk": "4097,333,2048,1,900",
         "h": 12, "hk": 4, "causal": True, "train": True},
        # training on packed images and clips, all heads
        {"name": "packed_train_clips", "op": "packed", "lq": "1560,7800,1560", "lk": "1560,7800,1560",
         "h": 12, "hk": 12, "causal": False, "train": True},
        # one short stream: latency
        {"name": "decode_one", "op": "decode", "lens": "300", "h": 12, "hk": 12, "page": 16},
        # a ragged batch with grouped heads; a fresh stream with nothing cached yet
        {"name": "decode_batch", "op": "decode", "lens": ",".join(str((i * 2657) % 8192) for i in range(48)),
         "h": 40, "hk": 8, "page": 64},
        # a few streams with whole videos behind them (21 x 45 x 80 and 21 x 30 x 52 tokens)
        {"name": "decode_long", "op": "decode", "lens": "75600,75600,32760,32760", "h": 12, "hk": 12, "page": 100},
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("rope", "packed", "packed", "decode"))
    if op == "rope":
        h, hk = rng.choice(((12, 12), (40, 40), (16, 4), (10, 2), (7, 7), (32, 1)))
        t, hh, ww = _log(rng, 1, 21), _log(rng, 1, 45), _log(rng, 1, 80)
        dtype = rng.choice(("bf16", "bf16", "fp32"))
        return {"op": "rope", "b": rng.choice((1, 1, 2, 3)) if h <= 16 else 1, "t": t, "hh": hh, "ww": ww, "h": h, "hk": hk,
                "pad": rng.choice((0, 0, _log(rng, 1, 300))), "dtype": dtype, "train": dtype == "bf16" and rng.random() < 0.4}
    if op == "packed":
        hk = rng.choice((1, 2, 3, 4, 12))
        h = hk * rng.choice((1, 3, 4) if hk < 12 else (1,))
        train, causal = rng.random() < 0.5, rng.random() < 0.6
        n = _log(rng, 1, 16)
        most = int(math.sqrt((2.0e9 if train else 3.0e9) / (n * h)))  # the longest of n padded to it
        top = _log(rng, 32, min(most, 12000))
        lk = [top] + [rng.choice((0, 1, _log(rng, 1, top), _log(rng, 1, top), rng.randint(1, top))) for _ in range(n - 1)]
        rng.shuffle(lk)
        kind = rng.choice(("same", "same", "prefix", "other"))
        lq = [x if kind == "same" else rng.randint(0, x) if kind == "prefix" else _log(rng, 1, top) for x in lk]
        if max(lq) == 0:
            lq[0] = 1
        return {"op": "packed", "lq": ",".join(map(str, lq)), "lk": ",".join(map(str, lk)), "h": h, "hk": hk, "causal": causal,
                "train": train}
    hk = rng.choice((1, 2, 4, 8, 12))
    h = hk * rng.choice((1, 2, 3, 5, 8, 16))
    b = _log(rng, 1, 64)
    top = _log(rng, 1, min(75600, int(1.2e6 / (b * hk)) + 1))
    lens = [rng.choice((top, rng.randint(0, top), rng.randint(0, top), _log(rng, 1, top))) for _ in range(b)]
    lens[rng.randrange(b)] = top
    return {"op": "decode", "lens": ",".join(map(str, lens)), "h": h, "hk": hk, "page": rng.choice((1, 7, 16, 32, 64, 100, 128, 256))}


def _lens(text):
    return [int(x) for x in text.split(",")]


# ------------------------------------------------------------------ inputs
def _rnd(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _frequencies(device):
    """(64,) fp64: the angle per unit of position of every pair."""
    return torch.cat([THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device=device) / d) for d in AXES])


def _offsets(lens):
    at = [0]
    for x in lens:
        at.append(at[-1] + x)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] == "rope":
        n = case["t"] * case["hh"] * case["ww"]
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        # where the clip's first frame stands in its video: another seed, another place
        first = int(torch.randint(0, MAX_POS - 128, (1,), generator=g, device="cuda"))
        i = torch.arange(n, device="cuda")
        pos = torch.stack((first + i // (case["hh"] * case["ww"]), i // case["ww"] % case["hh"], i % case["ww"]), 1)
        s["positions"] = torch.cat((pos, torch.full((case["pad"], 3), -1, device="cuda"))).to(torch.int32)
        a = torch.arange(MAX_POS, dtype=torch.float64, device="cuda")[:, None] * _frequencies("cuda")
        s["table"] = torch.stack((a.cos(), a.sin()), -1).float()  # (MAX_POS, 64, 2)
        shape = (case["b"], n + case["pad"])
        s["q"], s["k"] = _rnd(g, *shape, case["h"], D, dtype=dt), _rnd(g, *shape, case["hk"], D, dtype=dt)
        if case["train"]:
            s["gq"], s["gk"] = _rnd(g, *shape, case["h"], D, dtype=dt), _rnd(g, *shape, case["hk"], D, dtype=dt)
    elif case["op"] == "packed":
        lq, lk = _lens(case["lq"]), _lens(case["lk"])
        s["q"] = _rnd(g, sum(lq), case["h"], D)
        s["k"], s["v"] = _rnd(g, sum(lk), case["hk"], D), _rnd(g, sum(lk), case["hk"], D)
        s["q_offsets"], s["k_offsets"] = _offsets(lq), _offsets(lk)
        s["max_q"], s["max_k"] = max(lq), max(lk)
        if case["train"]:
            s["do"] = _rnd(g, sum(lq), case["h"], D)
    else:
        lens = _lens(case["lens"])
        per = [-(-x // case["page"]) for x in lens]
        width, total = max(1, max(per)), sum(per)
        pages = total + 3  # a few free pages
        s["q"] = _rnd(g, len(lens), case["h"], D)
        s["k_cache"] = _rnd(g, pages, case["page"], case["hk"], D)
        s["v_cache"] = _rnd(g, pages, case["page"], case["hk"], D)
        order = torch.randperm(pages, generator=g, device="cuda")[:total].to(torch.int32)  # as an allocator leaves them
        have = torch.arange(width, device="cuda")[None] < torch.tensor(per, device="cuda")[:, None]
        table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
        table[have] = order
        s["page_table"] = table
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------ plain forms
def _turn(x, positions, table, sign):
    at = positions.clamp(min=0).long()
    pair = torch.arange(D // 2, device=x.device)
    axis = (pair >= AXES[0] // 2).long() + (pair >= (AXES[0] + AXES[1]) // 2)
    cs = table[at[:, axis], pair]  # (s, 64, 2)
    still = (positions < 0).any(1)[:, None]
    cos = torch.where(still, 1.0, cs[..., 0])[:, None]
    sin = torch.where(still, 0.0, cs[..., 1])[:, None] * sign
    f = x.float()
    a, b = f[..., 0::2], f[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2).to(x.dtype)


def _padded(x, offsets, width):
    """(total, heads, D) -> fp32 (n, heads, width, D), zeros behind each sequence, and who is there (n, width)."""
    i = torch.arange(width, device=x.device)
    there = i[None] < (offsets[1:] - offsets[:-1])[:, None]
    at = torch.where(there, offsets[:-1, None].long() + i[None], 0)
    y = torch.where(there[..., None, None], x.float()[at], 0.0)
    return y.transpose(1, 2), there


def _packed_plain(s):
    h, hk, n = s["h"], s["hk"], s["q_offsets"].numel() - 1
    q, is_q = _padded(s["q"], s["q_offsets"], s["max_q"])
    k, is_k = _padded(s["k"], s["k_offsets"], s["max_k"])
    v, _ = _padded(s["v"], s["k_offsets"], s["max_k"])
    q = q.reshape(n, hk, h // hk, s["max_q"], D)
    seen = is_k[:, None, :]
    if s["causal"]:
        shift = (is_k.sum(1) - is_q.sum(1))[:, None, None]
        seen = seen & (torch.arange(s["max_k"], device=q.device)[None, None, :]
                       <= torch.arange(s["max_q"], device=q.device)[None, :, None] + shift)
    seen = seen[:, None, None]
    p = (q @ k[:, :, None].transpose(-1, -2)).mul_(SCALE).masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    some = total > 0
    p = p.div_(torch.where(some, total, 1.0))
    o = p @ v[:, :, None]
    lse = torch.where(some, top + torch.where(some, total, 1.0).log(), -math.inf)[..., 0]
    rows = is_q.nonzero(as_tuple=True)

    def pack(x):  # (n, hk, g, max_q, ...) -> (total, h, ...)
        return x.flatten(1, 2).transpose(1, 2)[rows]

    out = [pack(o).to(s["q"].dtype), pack(lse).T.contiguous()]
    if not s["train"]:
        return out
    do = _padded(s["do"], s["q_offsets"], s["max_q"])[0].reshape(n, hk, h // hk, s["max_q"], D)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = (do @ v[:, :, None].transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    dq = (ds @ k[:, :, None]) * SCALE
    dk = (ds.transpose(-1, -2) @ q).sum(2) * SCALE
    keys = is_k.nonzero(as_tuple=True)
    return [out[0], pack(dq).to(s["q"].dtype), dk.transpose(1, 2)[keys].to(s["k"].dtype), dv.transpose(1, 2)[keys].to(s["v"].dtype)]


def _decode_plain(s):
    b, h, hk, page = s["q"].shape[0], s["h"], s["hk"], s["page"]
    width = s["page_table"].shape[1] * page
    at = s["page_table"].long()
    k = s["k_cache"][at].float().reshape(b, width, hk, D)
    v = s["v_cache"][at].float().reshape(b, width, hk, D)
    q = s["q"].float().reshape(b, hk, h // hk, D)
    there = (torch.arange(width, device=q.device)[None] < s["lengths"][:, None])[:, None, None]
    p = (q @ k.permute(0, 2, 3, 1)).mul(SCALE).masked_fill(~there, -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = (p - top).exp()
    total = p.sum(-1, keepdim=True)
    some = total > 0
    o = (p @ v.transpose(1, 2)) / torch.where(some, total, 1.0)
    lse = torch.where(some, top + torch.where(some, total, 1.0).log(), -math.inf)
    return [o.reshape(b, h, D).to(s["q"].dtype), lse.reshape(b, h)]


# ------------------------------------------------------------------ one pass
def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["op"] == "rope":
        out = [_turn(s["q"], s["positions"], s["table"], 1.0), _turn(s["k"], s["positions"], s["table"], 1.0)]
        if s["train"]:
            out += [_turn(s["gq"], s["positions"], s["table"], -1.0), _turn(s["gk"], s["positions"], s["table"], -1.0)]
        return out
    return _packed_plain(s) if s["op"] == "packed" else _decode_plain(s)


def _run_own(s):
    if s["op"] == "rope":
        from wan_flash.rope import wan_flash_rope

        if not s["train"]:
            return list(wan_flash_rope(s["q"], s["k"], s["positions"], s["table"]))
        q, k = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
        yq, yk = wan_flash_rope(q, k, s["positions"], s["table"])
        return [yq.detach(), yk.detach(), *torch.autograd.grad((yq, yk), (q, k), (s["gq"], s["gk"]))]
    if s["op"] == "packed":
        from wan_flash.packed import wan_flash_attn_packed, wan_flash_packed_fwd

        if not s["train"]:
            return list(wan_flash_packed_fwd(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], causal=s["causal"]))
        q, k, v = (s[x].detach().requires_grad_() for x in ("q", "k", "v"))
        o = wan_flash_attn_packed(q, k, v, s["q_offsets"], s["k_offsets"], causal=s["causal"])
        return [o.detach(), *torch.autograd.grad(o, (q, k, v), s["do"])]
    from wan_flash.decode import wan_flash_decode

    return list(wan_flash_decode(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"]))


# ------------------------------------------------------------------ what a pass cannot do without
def _pairs(lq, lk, causal):
    """Query-key pairs that the masks leave."""
    if not causal:
        return sum(a * b for a, b in zip(lq, lk))
    n = 0
    for a, b in zip(lq, lk):
        first = b - a + 1  # keys that row 0 sees; row i sees first + i of them, at least none, at most b
        empty = min(a, max(0, -first))
        rows = a - empty
        n += rows * max(first, 0) + rows * (rows - 1) // 2
    return n


def work(case):
    if case["op"] == "rope":
        tokens = case["b"] * (case["t"] * case["hh"] * case["ww"] + case["pad"])
        size = 2 if case["dtype"] == "bf16" else 4
        passes = 2 if case["train"] else 1
        values = tokens * (case["h"] + case["hk"]) * D
        return {"bytes": passes * (2 * values * size) + 12 * (tokens // case["b"]), "flops": passes * 3 * values}
    if case["op"] == "packed":
        lq, lk = _lens(case["lq"]), _lens(case["lk"])
        rows, keys = sum(lq) * case["h"], sum(lk) * case["hk"]
        pairs = _pairs(lq, lk, case["causal"]) * case["h"]
        if not case["train"]:
            return {"bytes": rows * (2 * 256 + 4) + keys * 2 * 256, "flops": 4 * D * pairs}
        # q, do in; o, dq out; k, v in; dk, dv out; two products forward, five backward
        return {"bytes": rows * 4 * 256 + keys * 4 * 256, "flops": 14 * D * pairs}
    lens = _lens(case["lens"])
    return {"bytes": sum(lens) * case["hk"] * 512 + len(lens) * case["h"] * (512 + 4) + 4 * (len(lens) + sum(-(-x // case["page"]) for x in lens)),
            "flops": 4 * D * case["h"] * sum(lens)}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        f = _frequencies("cuda")
        pos = s["positions"].double()
        angle = torch.cat([pos[:, a:a + 1] * f[sum(AXES[:a]) // 2:sum(AXES[:a + 1]) // 2] for a in range(3)], 1)
        angle[(pos < 0).any(1)] = 0.0

        def turned(x, sign):
            z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], D // 2, 2))
            z = z * torch.polar(torch.ones_like(angle), sign * angle)[:, None]
            return torch.view_as_real(z).flatten(-2)

        return [turned(s["q"], 1), turned(s["k"], 1)] + ([turned(s["gq"], -1), turned(s["gk"], -1)] if case["train"] else [])
    if case["op"] == "packed":
        q, k, v = (s[x].double() for x in ("q", "k", "v"))
        group = case["h"] // case["hk"]
        o, lse = torch.zeros_like(q), torch.full((case["h"], q.shape[0]), -math.inf, dtype=torch.float64, device="cuda")
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        qa = ka = 0
        for a, b in zip(_lens(case["lq"]), _lens(case["lk"])):
            for h in range(case["h"] if a and b else 0):
                c = h // group
                x, y, z = q[qa:qa + a, h], k[ka:ka + b, c], v[ka:ka + b, c]
                w = x @ y.T / math.sqrt(D)
                if case["causal"]:
                    w = torch.where(torch.ones_like(w, dtype=torch.bool).tril(b - a), w, -math.inf)
                e = torch.logsumexp(w, 1)
                w = torch.where(e[:, None] == -math.inf, 0.0, (w - torch.where(e == -math.inf, 0.0, e)[:, None]).exp())
                r = w @ z
                o[qa:qa + a, h], lse[h, qa:qa + a] = r, e
                if case["train"]:
                    t = s["do"][qa:qa + a, h].double()
                    dv[ka:ka + b, c] += w.T @ t
                    u = w * (t @ z.T - (t * r).sum(1, keepdim=True)) / math.sqrt(D)
                    dq[qa:qa + a, h] = u @ y
                    dk[ka:ka + b, c] += u.T @ x
            qa, ka = qa + a, ka + b
        return [o, dq, dk, dv] if case["train"] else [o, lse]
    lens = _lens(case["lens"])
    o = torch.zeros(len(lens), case["h"], D, dtype=torch.float64, device="cuda")
    lse = torch.full((len(lens), case["h"]), -math.inf, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        if n:
            at = torch.arange(n, device="cuda")
            page = s["page_table"][i].long()[at // case["page"]]
            k = s["k_cache"][page, at % case["page"]].double().repeat_interleave(case["h"] // case["hk"], 1)
            v = s["v_cache"][page, at % case["page"]].double().repeat_interleave(case["h"] // case["hk"], 1)
            w = torch.einsum("hd,nhd->hn", s["q"][i].double(), k) / math.sqrt(D)
            lse[i] = torch.logsumexp(w, 1)
            o[i] = torch.einsum("hn,nhd->hd", w.softmax(1), v)
    return [o, lse]
