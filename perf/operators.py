"""Measured cases of the decoder operators: an embedding lookup with scaling
and its gradient by sorted ids, layer norm with its weight gradients, and
cross attention from option (or beam) queries to an encoder's states.

`run` computes each in its plain form with elementary torch operations, or,
where `own` is true, through ptcg_b200.ops.
"""
import functools
import math

import torch

own = False

DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5


@functools.lru_cache(None)
def _ops():
    import __graft_entry__
    __graft_entry__.load_package()
    import ptcg_b200.ops
    return ptcg_b200.ops


# ------------------------------------------------------------------- cases
def _embedding(name, n, vocab, width, table, out, grad, skew, pad):
    return {"name": name, "op": "embedding", "n": n, "vocab": vocab, "width": width,
            "table": table, "out": out, "grad": grad, "skew": skew, "pad": pad}


def _norm(name, rows, width, x, y, grad, res):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "x": x, "y": y,
            "grad": grad, "res": res}


def _cross(name, nseq, lq, lk, heads, kv, dh, dtype, mask, layout, grad):
    return {"name": name, "op": "cross", "nseq": nseq, "lq": lq, "lk": lk, "heads": heads,
            "kv": kv, "dh": dh, "dtype": dtype, "mask": mask, "layout": layout, "grad": grad}


def listed():
    return [
        # the 64 option cards of one decision, looked up while a game waits
        _embedding("embed_decision", 64, 4096, 128, "fp32", "bf16", False, True, False),
        # the card ids of a 16384-sample training minibatch (128 tokens each)
        # with the c0 card table: most slots hold the same few ids
        _embedding("embed_train_cards", 16384 * 128, 4096, 128, "fp32", "bf16", True, True, False),
        # text tokens: a wide table that most of the batch touches once, an
        # odd vocabulary, and a padding id that takes no gradient
        _embedding("embed_train_text", 32768, 65537, 1024, "bf16", "bf16", True, False, True),
        # one residual row of one decision
        _norm("norm_decision", 1, 256, "fp32", "bf16", False, False),
        # the trunk's norm over a 16384-sample minibatch of 129 rows: fp32
        # residual stream in, bf16 GEMM operand out, the residual's own
        # gradient added on the way back
        _norm("norm_train_trunk", 16384 * 129, 256, "fp32", "bf16", True, True),
        # a wide norm of odd size in bf16
        _norm("norm_train_odd", 4099, 5001, "bf16", "bf16", True, False),
        # four decisions, one query each, over one board's encoder rows
        _cross("cross_decision", 4, 1, 129, 8, 8, 32, "bf16", "keep", "rows", False),
        # one query per sequence over a long cache laid out by head, four
        # query heads to a key head, caches of unequal length
        _cross("cross_history", 8, 1, 65536, 16, 4, 128, "bf16", "len", "heads", False),
        # a 1024-row rollout: 64 options against 129 board rows
        _cross("cross_rollout", 1024, 64, 129, 8, 8, 32, "bf16", "keep", "rows", False),
        # an 8192-sample training minibatch of the same widths
        _cross("cross_train", 8192, 64, 129, 8, 8, 32, "bf16", "keep", "rows", True),
        # exact fp32 training with odd lengths
        _cross("cross_train_fp32", 512, 61, 186, 8, 8, 32, "fp32", "len", "rows", True),
        # long queries over long states, grouped heads of width 128
        _cross("cross_train_long", 2, 4101, 8191, 16, 4, 128, "bf16", "none", "rows", True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["embedding", "norm", "cross", "cross"])
    grad = rng.random() < 0.6
    if op == "embedding":
        width = _log(rng, 32, 2048)
        if rng.random() < 0.7:
            width = max(32, width // 8 * 8)
        n = min(_log(rng, 1, 16384 * 128), (1 << 28) // width)
        vocab = min(_log(rng, 64, 131072), (1 << 26) // width)
        case = _embedding("", n, vocab, width, rng.choice(["fp32", "bf16"]),
                          rng.choice(["fp32", "bf16"]), grad, rng.random() < 0.5,
                          rng.random() < 0.5)
    elif op == "norm":
        width = _log(rng, 32, 8192)
        if rng.random() < 0.7:
            width = max(32, width // 8 * 8)
        rows = min(_log(rng, 1, 16384 * 129), (1 << 28) // width)
        case = _norm("", rows, width, rng.choice(["fp32", "bf16"]), rng.choice(["fp32", "bf16"]),
                     grad, rng.random() < 0.5)
    else:
        dh = rng.choice([32, 32, 64, 128])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 1, 2, 4])
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        lq = 1 if rng.random() < 0.25 else _log(rng, 2, 4096)
        # with one key the query and key gradients are zero by cancellation,
        # and a relative distance from them says nothing
        lk = _log(rng, 64 if grad else 1, 65536)
        nseq = _log(rng, 1, 4096)
        # products of the largest listed case at most, a quarter of them in
        # fp32, and an eighth of its keys and queries
        most = (1 << 38) if dtype == "bf16" else (1 << 35)
        while nseq > 1 and (nseq * heads * dh * lq * lk > most or nseq * heads * lq * lk > (1 << 30)
                            or nseq * kv * lk * dh > (1 << 28) or nseq * heads * lq * dh > (1 << 27)):
            nseq = (nseq + 1) // 2
        while lk > 64 and (nseq * heads * dh * lq * lk > most or nseq * heads * lq * lk > (1 << 30)):
            lk = (lk + 1) // 2
        case = _cross("", nseq, lq, lk, heads, kv, dh, dtype, rng.choice(["none", "keep", "len"]),
                      rng.choice(["rows", "heads"]), grad)
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)
    return g


def prepare(case, seed):
    g = _gen(seed)

    def rand(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    def unif(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = {"case": case}
    if case["op"] == "embedding":
        n, vocab, width = case["n"], case["vocab"], case["width"]
        u = unif(n).double()
        if case["skew"]:       # frequencies falling as 1 / rank, a few ids in most places
            ids = torch.exp(u * math.log(vocab)).long() - 1
        else:
            ids = (u * vocab).long()
        s["ids"] = ids.clamp_(0, vocab - 1).int()
        s["table"] = rand(vocab, width, dtype=DT[case["table"]])
        s["scale"] = math.sqrt(width)
        if case["grad"]:
            s["dout"] = rand(n, width, dtype=DT[case["out"]])
        return s
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        x = rand(rows, width)
        # residual rows differ in size and carry an offset
        x.mul_(0.25 + 2 * unif(rows, 1)).add_(rand(rows, 1))
        s["x"] = x.to(DT[case["x"]])
        s["gamma"] = 1 + 0.1 * rand(width)
        s["beta"] = 0.1 * rand(width)
        if case["grad"]:
            s["dy"] = rand(rows, width, dtype=DT[case["y"]])
            s["dres"] = rand(rows, width, dtype=DT[case["x"]]) if case["res"] else None
        return s
    nseq, lq, lk, dt = case["nseq"], case["lq"], case["lk"], DT[case["dtype"]]
    heads, kv, dh = case["heads"], case["kv"], case["dh"]
    s["q"] = rand(nseq, lq, heads, dh, dtype=dt)
    if case["layout"] == "heads":
        s["k"] = rand(nseq, kv, lk, dh, dtype=dt).transpose(1, 2)
        s["v"] = rand(nseq, kv, lk, dh, dtype=dt).transpose(1, 2)
    else:
        s["k"] = rand(nseq, lk, kv, dh, dtype=dt)
        s["v"] = rand(nseq, lk, kv, dh, dtype=dt)
    s["keep"] = s["kv_len"] = None
    if case["mask"] == "keep":         # padded tails and holes; the first row always stays
        fill = (0.3 + 0.7 * unif(nseq, 1)) * lk
        keep = (torch.arange(lk, device="cuda") < fill) & (unif(nseq, lk) < 0.9)
        keep[:, 0] = True
        s["keep"] = keep
    elif case["mask"] == "len":        # unequal lengths; a short one may be empty
        n = (unif(nseq) * (lk + 1)).int().clamp_(max=lk)
        s["kv_len"] = torch.where(n == 1, min(2, lk), n).int()
    if case["grad"]:
        s["dout"] = rand(nseq, lq, heads, dh, dtype=dt)
    return s


# ------------------------------------------------------------- plain forms
def _plain_embedding(s):
    case = s["case"]
    ids, scale = s["ids"].long(), s["scale"]
    live = (ids != 0) if case["pad"] else torch.ones_like(ids, dtype=torch.bool)
    out = torch.where(live[:, None], s["table"][ids].float() * scale, 0.0).to(DT[case["out"]])
    if not case["grad"]:
        return out
    # 64 bits: one id can hold a million places
    d = torch.where(live[:, None], s["dout"].double(), 0.0)
    acc = torch.zeros(case["vocab"], case["width"], dtype=torch.float64, device=d.device)
    acc.index_add_(0, ids, d)
    return out, (acc * scale).float()


def _plain_norm(s):
    case = s["case"]
    x = s["x"].float()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS)
    h = c * rstd
    y = (h * s["gamma"] + s["beta"]).to(DT[case["y"]])
    if not case["grad"]:
        return y
    dy = s["dy"].float()
    gy = dy * s["gamma"]
    dx = rstd * (gy - gy.mean(-1, keepdim=True) - h * (gy * h).mean(-1, keepdim=True))
    if s["dres"] is not None:
        dx = dx + s["dres"].float()
    return (y, mean[:, 0], rstd[:, 0], dx.to(DT[case["x"]]),
            (dy * h).sum(0, dtype=torch.float64).float(), dy.sum(0, dtype=torch.float64).float())


def _plain_cross(s):
    case = s["case"]
    nseq, lq, lk = case["nseq"], case["lq"], case["lk"]
    kv, group, dh, dt = case["kv"], case["heads"] // case["kv"], case["dh"], DT[case["dtype"]]
    scale = 1 / math.sqrt(dh)
    # the query heads of one key head are its rows: [nseq, kv, group * lq, dh]
    rows = lambda t: t.float().view(nseq, lq, kv, group, dh).permute(0, 2, 3, 1, 4).reshape(  # noqa: E731
        nseq, kv, group * lq, dh)
    back = lambda t: t.view(nseq, kv, group, lq, dh).permute(0, 3, 1, 2, 4).reshape(  # noqa: E731
        nseq, lq, kv * group, dh).to(dt)
    keys = lambda t: t.float().transpose(1, 2)  # noqa: E731
    q, k, v = rows(s["q"]), keys(s["k"]), keys(s["v"])
    sc = torch.matmul(q, k.transpose(-1, -2)) * scale
    if s["keep"] is not None:
        sc = torch.where(s["keep"][:, None, None, :], sc, -math.inf)
    if s["kv_len"] is not None:
        at = torch.arange(lk, device=sc.device)
        sc = torch.where((at < s["kv_len"][:, None])[:, None, None, :], sc, -math.inf)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(sc - m)
    del sc
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    del e
    lse = (m + torch.log(total)).view(nseq, kv * group, lq)
    o = torch.matmul(p, v)
    if not case["grad"]:
        return back(o), lse
    do = rows(s["dout"])
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, v.transpose(-1, -2))
    ds = p * (ds - (do * o).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(-1, -2), q) * scale
    return back(o), lse, back(dq), dk.transpose(1, 2).to(dt), dv.transpose(1, 2).to(dt)


# --------------------------------------------------------- the framework's
def _own_embedding(s):
    case, ops = s["case"], _ops()
    pad = 0 if case["pad"] else None
    out = ops.embedding(s["table"], s["ids"], scale=s["scale"], pad_id=pad,
                        out_dtype=DT[case["out"]])
    if not case["grad"]:
        return out
    return out, ops.embedding_backward(s["dout"], s["ids"], case["vocab"], scale=s["scale"],
                                       pad_id=pad)


def _own_norm(s):
    case, ops = s["case"], _ops()
    y, mean, rstd = ops.layer_norm(s["x"], s["gamma"], s["beta"], eps=EPS,
                                   out_dtype=DT[case["y"]], stats=case["grad"])
    if not case["grad"]:
        return y
    dx, dgamma, dbeta = ops.layer_norm_backward(s["dy"], s["x"], s["gamma"], mean, rstd,
                                                dres=s["dres"])
    return y, mean, rstd, dx, dgamma, dbeta


def _own_cross(s):
    case, ops = s["case"], _ops()
    mask = {"keep": s["keep"], "kv_len": s["kv_len"]}
    out, lse = ops.cross_attention(s["q"], s["k"], s["v"], **mask)
    if not case["grad"]:
        return out, lse
    return (out, lse, *ops.cross_attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse,
                                                    **mask))


def run(state):
    op = state["case"]["op"]
    if op == "embedding":
        return _own_embedding(state) if own else _plain_embedding(state)
    if op == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own_cross(state) if own else _plain_cross(state)


# -------------------------------------------------------------------- work
def _size(dtype):
    return 4 if dtype == "fp32" else 2


def work(case):
    if case["op"] == "embedding":
        n, w, v = case["n"], case["width"], case["vocab"]
        b = 4 * n + n * w * _size(case["out"]) + min(n, v) * w * _size(case["table"])
        f = n * w
        if case["grad"]:
            b += n * w * _size(case["out"]) + 4 * v * w
            f += n * w
        return {"bytes": b, "flops": f}
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        xs, ys = _size(case["x"]), _size(case["y"])
        b, f = n * (xs + ys) + 8 * case["width"], 8 * n
        if case["grad"]:
            b += n * (ys + xs + (xs if case["res"] else 0)) + 8 * case["width"] + 8 * case["rows"]
            f += 14 * n
        return {"bytes": b, "flops": f}
    kept = 0.5 if case["mask"] == "len" else 1.0       # mean share of the keys that count
    size = _size(case["dtype"])
    rows = case["nseq"] * case["lq"] * case["heads"]
    qb = rows * case["dh"] * size
    kb = case["nseq"] * case["lk"] * case["kv"] * case["dh"] * size
    f = 4.0 * rows * case["lk"] * kept * case["dh"]
    b = 2 * qb + 2 * kb * kept + 4 * rows
    if case["grad"]:
        b += 2 * qb + 2 * kb
        f *= 3.5
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------- exact
def _exact_embedding(s):
    case = s["case"]
    ids = s["ids"].long()
    out = s["table"].double()[ids] * s["scale"]
    if case["pad"]:
        out[ids == 0] = 0
    if not case["grad"]:
        return out
    # running sums over the places in order of their ids
    order = torch.argsort(ids, stable=True)
    run_ = torch.cumsum(s["dout"].double()[order], 0)
    run_ = torch.cat([torch.zeros_like(run_[:1]), run_])
    bounds = torch.searchsorted(ids[order].contiguous(),
                                torch.arange(case["vocab"] + 1, device=ids.device))
    grad = (run_[bounds[1:]] - run_[bounds[:-1]]) * s["scale"]
    if case["pad"]:
        grad[0] = 0
    return out, grad


def _exact_norm(s):
    case = s["case"]
    x, gamma = s["x"].double(), s["gamma"].double()
    var, mean = torch.var_mean(x, -1, correction=0)
    rstd = (var + EPS).rsqrt()
    h = (x - mean[:, None]) * rstd[:, None]
    del x
    y = torch.addcmul(s["beta"].double(), h, gamma)
    if not case["grad"]:
        return y
    dy = s["dy"].double()
    dbeta, dgamma = dy.sum(0), torch.einsum("rw,rw->w", dy, h)
    dy = dy * gamma
    w = case["width"]
    dx = dy - dy.sum(-1, keepdim=True) / w - h * (torch.einsum("rw,rw->r", dy, h) / w)[:, None]
    dx *= rstd[:, None]
    if s["dres"] is not None:
        dx += s["dres"].double()
    return y, mean, rstd, dx, dgamma, dbeta


def _exact_cross(s):
    case = s["case"]
    nseq, lq, lk, heads, dh = (case[k] for k in ("nseq", "lq", "lk", "heads", "dh"))
    group = heads // case["kv"]
    grad = case["grad"]
    new = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)  # noqa: E731
    out, lse = new(s["q"]), torch.zeros(nseq, heads, lq, dtype=torch.float64, device="cuda")
    dq, dk, dv = (new(s[n]) for n in ("q", "k", "v")) if grad else (None, None, None)
    live = torch.ones(nseq, lk, dtype=torch.bool, device="cuda")
    if s["keep"] is not None:
        live &= s["keep"]
    if s["kv_len"] is not None:
        live &= torch.arange(lk, device="cuda")[None] < s["kv_len"][:, None]
    step = max(1, (1 << 27) // (lq * lk))        # sequences at a time, one head each
    for h in range(heads):
        c = h // group
        for a in range(0, nseq, step):
            b = min(nseq, a + step)
            q, k, v = s["q"][a:b, :, h].double(), s["k"][a:b, :, c].double(), s["v"][a:b, :, c].double()
            sc = torch.einsum("nid,njd->nij", q, k) / math.sqrt(dh)
            sc.masked_fill_(~live[a:b, None, :], -math.inf)
            lse[a:b, h] = torch.logsumexp(sc, -1)
            p = torch.exp(sc - lse[a:b, h, :, None])
            p[~live[a:b].any(-1)] = 0
            o = torch.einsum("nij,njd->nid", p, v)
            out[a:b, :, h] = o
            if grad:
                do = s["dout"][a:b, :, h].double()
                dv[a:b, :, c] += torch.einsum("nij,nid->njd", p, do)
                p *= torch.einsum("nid,njd->nij", do, v) - torch.einsum("nid,nid->ni", do, o)[..., None]
                dq[a:b, :, h] = torch.einsum("nij,njd->nid", p, k) / math.sqrt(dh)
                dk[a:b, :, c] += torch.einsum("nij,nid->njd", p, q) / math.sqrt(dh)
    return (out, lse, dq, dk, dv) if grad else (out, lse)


def exact(case, seed):
    s = prepare(case, seed)
    return {"embedding": _exact_embedding, "norm": _exact_norm, "cross": _exact_cross}[case["op"]](s)
