"""The decoder operators' formulas in 64 bits, with a bound on how far an
fp32-accumulating implementation may be from them, element by element.

u = 2^-24 is half a step of fp32.  A sum of n terms in any order is off by at
most n u times the sum of their magnitudes (first order); a product adds one
u; a rounding to bf16 adds 2^-8 of the value.  ex2.approx and rsqrt are
allowed 2^-21 (a few units of the last place)."""
import math

import torch

U = 2.0 ** -24
HALF = {torch.float64: 0.0, torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
FN = 2.0 ** -21


def within(got, want, bound, what=""):
    got, want = got.double().cpu(), want.double().cpu()
    bound = bound.double().cpu() + 1e-37                 # results below fp32's range
    same = (got == want) | (got.isnan() & want.isnan())
    err = torch.where(same, torch.zeros_like(want), (got - want).abs())
    bad = ~(err <= bound)
    if bad.any():
        i = int((err / bound).nan_to_num(math.inf).flatten().argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst at {i}: "
                             f"{got.flatten()[i]:.9g} for {want.flatten()[i]:.9g}, "
                             f"bound {bound.flatten()[i]:.3g}")


# -------------------------------------------------------------- embedding
def embedding(table, ids, scale, pad, out_dtype):
    i = ids.long().clamp(0, table.shape[0] - 1)
    y = table.double()[i] * scale
    if pad is not None:
        y[ids == pad] = 0
    return y, y.abs() * (2 * U + HALF[out_dtype])


def embedding_grad(dout, ids, vocab, scale, pad):
    d = dout.double().reshape(-1, dout.shape[-1])
    i = ids.long().reshape(-1)
    live = torch.ones_like(i, dtype=torch.bool) if pad is None else i != pad
    i = i.clamp(0, vocab - 1)[live]
    d = d[live]
    z = torch.zeros(vocab, d.shape[1], dtype=torch.float64, device=d.device)
    g, mag = z.clone().index_add_(0, i, d), z.index_add_(0, i, d.abs())
    cnt = torch.bincount(i, minlength=vocab).double()[:, None]
    return g * scale, mag * abs(scale) * (cnt + 3) * U


# ------------------------------------------------------------- layer norm
def norm(x, gamma, beta, eps):
    """dict of the forward's values and bounds"""
    x = x.double()
    w = x.shape[-1]
    g = torch.ones(w, dtype=torch.float64, device=x.device) if gamma is None else gamma.double()
    b = torch.zeros(w, dtype=torch.float64, device=x.device) if beta is None else beta.double()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    var = (c * c).mean(-1, keepdim=True)
    rstd = (var + eps) ** -0.5
    h = c * rstd
    depth = w / 16 + 24                   # additions a term goes through at most
    e_mean = (depth + 2) * U * x.abs().mean(-1, keepdim=True)
    # the variance about the computed mean gains e_mean^2; x - mean is off by u
    # of itself and e_mean
    e_var = (depth + 4) * U * var + e_mean ** 2
    rel_r = 0.5 * e_var / (var + eps) + FN
    e_h = rstd * e_mean + h.abs() * (rel_r + 3 * U)
    y = h * g + b
    return {"x": x, "g": g, "mean": mean, "rstd": rstd, "h": h, "y": y, "e_mean": e_mean,
            "e_rstd": rstd * rel_r, "rel_r": rel_r, "e_h": e_h, "depth": depth,
            "e_y": g.abs() * e_h + 2 * U * ((h * g).abs() + b.abs())}


def norm_grad(f, dy, dres, dtype):
    dy = dy.double()
    g, h, r, w = dy * f["g"], f["h"], f["rstd"], dy.shape[-1]
    m1, m2 = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    a1, a2 = g.abs().mean(-1, keepdim=True), (g * h).abs().mean(-1, keepdim=True)
    dx = r * (g - m1 - h * m2)
    k = (f["depth"] + 8) * U
    e_m2 = k * a2 + (g.abs() * f["e_h"]).mean(-1, keepdim=True)
    e = r * (4 * U * (g.abs() + a1 + h.abs() * a2) + k * a1 + f["e_h"] * a2 + h.abs() * e_m2)
    e = e + f["rel_r"] * r * (g - m1 - h * m2).abs()
    if dres is not None:
        dx = dx + dres.double()
        e = e + 2 * U * (dx.abs() + dres.double().abs())
    e = e + HALF[dtype] * dx.abs()
    dims = tuple(range(dy.dim() - 1))
    n = dy[..., 0].numel()
    dg, db = (dy * h).sum(dims), dy.sum(dims)
    e_dg = (n + 4) * U * (dy * h).abs().sum(dims) + (dy.abs() * f["e_h"]).sum(dims)
    return dx, e, dg, e_dg, db, (n + 4) * U * dy.abs().sum(dims)


# -------------------------------------------------------- cross attention
def live_keys(nseq, lk, keep, kv_len, device):
    live = torch.ones(nseq, lk, dtype=torch.bool, device=device)
    if keep is not None:
        live &= keep.bool()
    if kv_len is not None:
        live &= torch.arange(lk, device=device)[None] < kv_len[:, None]
    return live


def cross(q, k, v, keep=None, kv_len=None, scale=None, dout=None):
    """dict of out, lse (, dq, dk, dv) and their bounds e_*"""
    dt = q.dtype
    op = HALF[dt] if dt == torch.bfloat16 else 0.0        # P and dS rounded as operands
    nseq, lq, heads, dh = q.shape
    lk, kvh = k.shape[1], k.shape[2]
    grp = heads // kvh
    scale = dh ** -0.5 if scale is None else scale
    live = live_keys(nseq, lk, keep, kv_len, q.device)
    kz = torch.where(live[:, :, None, None], k.double(), 0.0).repeat_interleave(grp, 2)
    vz = torch.where(live[:, :, None, None], v.double(), 0.0).repeat_interleave(grp, 2)
    qd = q.double()
    dot = lambda a, b: torch.einsum("nihd,njhd->nhij", a, b)     # noqa: E731
    s = (dot(qd, kz) * scale).masked_fill(~live[:, None, None, :], -math.inf)
    has = live.any(-1)[:, None, None]
    m = torch.where(has, s.amax(-1) if lk else torch.zeros(nseq, heads, lq, dtype=torch.float64,
                                                           device=q.device), 0.0)
    e = torch.exp(s - m[..., None])
    tot = e.sum(-1)
    p = e / torch.where(tot == 0, 1.0, tot)[..., None]
    lse = m + torch.log(tot)
    # a score is off by the dot product's rounding and, in the exponent's
    # argument, by a few u of its own size
    e_s = (dh + 6) * U * dot(qd.abs(), kz.abs()) * scale
    e_s = (e_s + 4 * U * torch.where(live[:, None, None, :], s, 0.0).abs()).amax(-1) if lk else 0 * m
    e_s = e_s + 4 * U * m.abs()
    e_p = (2 * e_s + 4 * FN + (lk + 8) * U)[..., None]
    out = torch.einsum("nhij,njhd->nihd", p, vz)
    up = lambda t: t.transpose(1, 2)[..., None]                  # noqa: E731
    pv = torch.einsum("nhij,njhd->nihd", p, vz.abs())
    e_out = pv * up(e_p[..., 0] + op + (lk + 8) * U) + HALF[dt] * out.abs()
    r = {"out": out, "lse": lse, "e_out": e_out,
         "e_lse": e_s + 2 * FN + (lk + 8) * U + 4 * U * lse.abs().nan_to_num(posinf=0.0)}
    if dout is None:
        return r
    do = dout.double()
    dp = dot(do, vz)
    delta = (do * out).sum(-1).transpose(1, 2)[..., None]
    e_delta = ((do.abs() * e_out).sum(-1) + (dh + 4) * U * (do * out).abs().sum(-1))
    e_delta = e_delta.transpose(1, 2)[..., None]
    ds = p * (dp - delta)
    e_ds = ds.abs() * (e_p + op + 2 * U) + p * ((dh + 4) * U * dot(do.abs(), vz.abs()) + e_delta)
    r["dq"] = torch.einsum("nhij,njhd->nihd", ds, kz) * scale
    r["e_dq"] = (torch.einsum("nhij,njhd->nihd", e_ds + (lk + 8) * U * ds.abs(), kz.abs()) * scale
                 + HALF[dt] * r["dq"].abs())
    fold = lambda t: t.view(nseq, lk, kvh, grp, dh).sum(3)       # noqa: E731
    rows = lq * grp
    r["dk"] = fold(torch.einsum("nhij,nihd->njhd", ds, qd) * scale)
    r["e_dk"] = (fold(torch.einsum("nhij,nihd->njhd", e_ds + (rows + 8) * U * ds.abs(), qd.abs()))
                 * scale + HALF[dt] * r["dk"].abs())
    r["dv"] = fold(torch.einsum("nhij,nihd->njhd", p, do))
    r["e_dv"] = (fold(torch.einsum("nhij,nihd->njhd", p * (e_p + op + (rows + 8) * U), do.abs()))
                 + HALF[dt] * r["dv"].abs())
    return r
