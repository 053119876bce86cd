"""Softmax attention of one sequence in 64 bits, with grouped heads, causal or
not, and the error bounds of a kernel that holds scores, sums and O in fp32,
rounds the probabilities (and in the backward dS) to bf16 for the tensor
cores, and rounds every output once to bf16.

Rounding to nearest bf16 is off by at most U = 2^-8 of the value.  Scores are
sums of 128 fp32 products, off by at most 128 * 2^-23 * sum|q k| (the factor
2 of 2^-23 over the half step 2^-24 allows truncating accumulation); exp2 and
the running rescales add a few 2^-22.
"""

import math

import torch

U = 2.0 ** -8          # half a bf16 step
E32 = 2.0 ** -23       # an fp32 step
SCALE = 1.0 / math.sqrt(128)


def visible(lq, lk, causal, device):
    if not causal:
        return torch.ones(lq, lk, dtype=torch.bool, device=device)
    i = torch.arange(lq, device=device)[:, None]
    return torch.arange(lk, device=device)[None] <= i + lk - lq


def attn64(q, k, v, causal=False):
    """q (lq, h, 128), k, v (lk, h_kv, 128) -> o, lse (h, lq) and their bounds o_tol, lse_tol, and p (h, lq, lk)."""
    g = q.shape[1] // k.shape[1]
    q, k, v = (x.double().transpose(0, 1) for x in (q, k, v))
    k, v = k.repeat_interleave(g, 0), v.repeat_interleave(g, 0)
    lq, lk = q.shape[1], k.shape[1]
    see = visible(lq, lk, causal, q.device)
    s = torch.where(see, (q @ k.transpose(1, 2)) * SCALE, -math.inf)
    lse = torch.logsumexp(s, -1) if lk else torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    some = lse > -math.inf
    p = torch.where(some[..., None], (s - torch.where(some, lse, 0.0)[..., None]).exp(), 0.0)
    o = p @ v
    # error of a row's exponents: its largest score error (nats) plus exp2 / rescale roundings
    mass = torch.where(see, q.abs() @ k.abs().transpose(1, 2), 0.0) * SCALE
    es = 128 * E32 * (mass.amax(-1) if lk else torch.zeros_like(lse)) + 8 * E32
    spread = p @ v.abs()
    o_tol = (U + 4 * es[..., None] + lk * E32) * spread + U * (o.abs() + 2 * U * spread)
    lse_tol = es + (lk + 4) * E32 + 4 * E32 * torch.where(some, lse.abs(), 0.0)
    return {"o": o.transpose(0, 1), "lse": lse, "o_tol": o_tol.transpose(0, 1), "lse_tol": lse_tol, "p": p, "es": es}


def assert_close(got, want, tol, tag):
    got = got.double()
    assert got.shape == want.shape, (tag, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.where(fine, torch.zeros_like(got), got), torch.where(fine, torch.zeros_like(want), want)), \
        f"{tag}: infinities differ"
    over = torch.where(fine, (got - want).abs() - tol, torch.full_like(want, -1.0))
    over = torch.where(torch.isfinite(over), over, torch.full_like(over, math.inf))
    assert over.numel() == 0 or over.max().item() <= 0, \
        f"{tag}: off by {over.max().item():.3e} more than allowed, at {int(over.argmax())}"


def grads64(q, k, v, do, causal=False, residual=False):
    """dq, dk, dv of o = attention(q, k, v) given do, by the formulas in 64 bits, with their bounds.

    Errors of a kernel, entry by entry: P off by e = 4 es relative (its exponent: score and lse) and rounded to bf16
    (U) before dV = P^T do; dP = do v^T an fp32 sum; D = rowsum(o do) from the o that was rounded
    (o_tol; with its residual only o's error before that rounding, and its square); dS = P (dP -
    D) rounded to bf16 (U) before dQ and dK; fp32 sums over rows or keys; one rounding of the result."""
    r = attn64(q, k, v, causal)
    g, lq, lk = q.shape[1] // k.shape[1], q.shape[0], k.shape[0]
    x, y, z, t = (a.double().transpose(0, 1) for a in (q, k, v, do))
    y, z = y.repeat_interleave(g, 0), z.repeat_interleave(g, 0)
    p, o, o_tol = r["p"], r["o"].transpose(0, 1), r["o_tol"].transpose(0, 1)
    if residual:
        o_tol = o_tol - U * o.abs() + U * U * (o.abs() + o_tol)
    e = 4 * r["es"][..., None] + 16 * E32
    dp = t @ z.transpose(1, 2)
    delta = (t * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dp_err = 128 * E32 * (t.abs() @ z.abs().transpose(1, 2))
    delta_err = (o_tol * t.abs()).sum(-1, keepdim=True) + 128 * E32 * (t * o).abs().sum(-1, keepdim=True)
    ds_err = (U + (1 + U) * e) * ds.abs() + (1 + U) * p * (dp_err + delta_err)
    rows = (lq + lk) * E32
    out = {}
    p_err = (U + (1 + U) * e) * p
    out["dv"] = p.transpose(1, 2) @ t, (p_err + rows * p).transpose(1, 2) @ t.abs()
    out["dq"] = ds @ y * SCALE, (ds_err + rows * ds.abs()) @ y.abs() * SCALE
    out["dk"] = ds.transpose(1, 2) @ x * SCALE, (ds_err + rows * ds.abs()).transpose(1, 2) @ x.abs() * SCALE
    for name, (want, tol) in out.items():
        want, tol = want.transpose(0, 1), tol.transpose(0, 1)
        if name != "dq":  # the q heads of a group share the key-value head
            want, tol = (a.unflatten(1, (a.shape[1] // g, g)).sum(2) for a in (want, tol))
        out[name] = want, tol + U * (want.abs() + tol) + E32 * want.abs()
    return out
