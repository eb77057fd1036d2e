"""The decoder operators on the GPU against their formulas in 64 bits, inside
bounds that count the roundings (ops_reference.py), at the sizes, masks,
strides and calls where they can go wrong."""
import itertools
import math

import pytest
import torch

import ops_reference as ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops(pkg):
    import ptcg_b200.ops
    return ptcg_b200.ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


# -------------------------------------------------------------- embedding
@pytest.mark.parametrize("td,od", list(itertools.product([F32, BF16], repeat=2)))
@pytest.mark.parametrize("n,vocab,width", [(1, 1, 1), (3, 7, 8), (64, 4096, 128), (1000, 17, 33),
                                           (257, 50, 1032), (5, 9, 2049)])
def test_embedding_forward(ops, td, od, n, vocab, width):
    g = gen(n + width)
    table = rand(g, vocab, width, dtype=td)
    ids = torch.randint(-3, vocab + 3, (n,), generator=g, device="cuda", dtype=torch.int32)
    for pad in (None, 0):
        got = ops.embedding(table, ids, scale=1.7, pad_id=pad, out_dtype=od)
        scale = float(torch.tensor(1.7, dtype=F32))
        want, bound = ref.embedding(table, ids, scale, pad, od)
        assert got.dtype == od and got.shape == (n, width)
        ref.within(got, want, bound)


def test_embedding_forward_views(ops):
    g = gen(1)
    ids = torch.randint(0, 20, (2, 3, 5), generator=g, device="cuda", dtype=torch.int32)
    for table in (rand(g, 20, 72)[:, 8:40], rand(g, 20, 41)[:, 3:36], rand(g, 33, 20).t(),
                  rand(g, 20, 40, dtype=BF16)[:, 1:33]):
        got = ops.embedding(table, ids, scale=0.5)
        want, bound = ref.embedding(table, ids, 0.5, None, table.dtype)
        ref.within(got, want, bound)
    assert ops.embedding(rand(g, 4, 8), ids[:0]).shape == (0, 3, 5, 8)


GRADS = [  # n, vocab, width, how the ids fall
    (1, 1, 1, "one"), (1, 300, 8, "any"), (7, 3, 33, "any"), (64, 4096, 128, "any"),
    (31, 5, 40, "one"), (4095, 257, 8, "any"), (4097, 255, 64, "skew"), (8192, 256, 16, "one"), (8193, 600, 12, "any"), (16385, 600, 12, "skew"),
    (5000, 65537, 24, "any"), (3000, 70000, 9, "skew"), (20000, 40, 136, "skew"),
    (12289, 11, 7, "skew"), (2500, 4000, 520, "any"), (700001, 1000, 8, "skew"),
    (611000, 3, 1, "any"), (1024, 70000, 8, "any"), (1025, 300, 130, "skew"), (3000, 50, 301, "any")]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,vocab,width,how", GRADS)
def test_embedding_gradient(ops, dtype, n, vocab, width, how):
    g = gen(n + vocab)
    if how == "one":
        ids = torch.full((n,), vocab // 2, device="cuda", dtype=torch.int32)
    elif how == "any":
        ids = torch.randint(-2, vocab + 2, (n,), generator=g, device="cuda", dtype=torch.int32)
    else:
        u = torch.rand(n, generator=g, device="cuda")
        ids = (torch.exp(u * math.log(vocab)).int() - 1).clamp(0, vocab - 1)
    dout = rand(g, n, width, dtype=dtype)
    for pad in (None, vocab // 2):
        want, bound = ref.embedding_grad(dout, ids, vocab, 1.5, pad)
        got = ops.embedding_backward(dout, ids, vocab, scale=1.5, pad_id=pad)
        ref.within(got, want, bound, f"pad {pad}")
        again = ops.embedding_backward(dout, ids, vocab, scale=1.5, pad_id=pad)
        assert torch.equal(got, again)                     # no order that depends on scheduling
        base = rand(g, vocab, width)
        acc = ops.embedding_backward(dout, ids, vocab, scale=1.5, pad_id=pad, dtable=base.clone(),
                                     accumulate=True)
        ref.within(acc, base.double() + want, bound + 2 * ref.U * (base.double().abs() + want.abs()))
        rows = torch.unique(ids[ids != pad] if pad is not None else ids).long().clamp(0, vocab - 1)
        still = torch.ones(vocab, dtype=torch.bool, device="cuda")
        still[rows] = False
        assert torch.equal(acc[still], base[still])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,vocab,width,how", [
    (9000, 2, 40, "any"), (300001, 5, 24, "any"), (605000, 70000, 3, "skew"), (620000, 70000, 8, "skew"),
    (700001, 1000, 8, "skew"), (1212417, 3, 1, "any"), (1300001, 4096, 8, "skew"), (1 << 21, 1, 16, "any"),
    (1 << 21, 4096, 40, "skew")])
def test_embedding_gradient_exact_sums(ops, dtype, n, vocab, width, how):
    """Whole numbers of -3 to 3, whose sums stay below 2^24 and so are exact in
    fp32 in any order: not one place of a million may be lost or counted
    twice.  On both sides of the sort's tile sizes."""
    g = gen(n)
    if how == "any":
        ids = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    else:
        ids = (torch.exp(torch.rand(n, generator=g, device="cuda") * math.log(vocab)).int() - 1).clamp(0, vocab - 1)
    dout = torch.randint(-3, 4, (n, width), generator=g, device="cuda").to(dtype)
    want = torch.zeros(vocab, width, dtype=torch.float64, device="cuda").index_add_(0, ids.long(), dout.double())
    assert want.abs().max() * 4 < 2 ** 24 and 3 * n < 2 ** 24
    got = ops.embedding_backward(dout, ids, vocab, scale=4.0)
    assert torch.equal(got.double(), 4 * want)
    pad = vocab // 3
    base = torch.randint(-99, 99, (vocab, width), generator=g, device="cuda").float()
    acc = ops.embedding_backward(dout, ids, vocab, pad_id=pad, dtable=base.clone(), accumulate=True)
    want[pad] = 0
    assert torch.equal(acc.double(), base.double() + want)


def test_embedding_gradient_views(ops):
    g = gen(3)
    ids = torch.randint(0, 50, (6, 100), generator=g, device="cuda", dtype=torch.int32)
    big = rand(g, 6, 100, 80, dtype=BF16)
    for dout in (big[..., 8:72], big[..., 3:68], big[:, :, :64].transpose(0, 1).transpose(0, 1),
                 big[:1, :1, :32].expand(6, 100, 32)):
        width = dout.shape[-1]
        want, bound = ref.embedding_grad(dout, ids, 50, 1.0, None)
        ref.within(ops.embedding_backward(dout, ids, 50), want, bound)
        frame = torch.full((50, width + 8), 7.0, device="cuda")
        got = ops.embedding_backward(dout, ids, 50, dtable=frame[:, 4:width + 4])
        ref.within(got, want, bound)
        assert (frame[:, :4] == 7).all() and (frame[:, width + 4:] == 7).all()
    none = ops.embedding_backward(big[:0], ids[:0], 50)
    assert none.shape == (50, 80) and (none == 0).all()
    keep = torch.ones(50, 80, device="cuda")
    assert (ops.embedding_backward(big[:0], ids[:0], 50, dtable=keep, accumulate=True) == 1).all()


def test_embedding_padding_may_hold_anything(ops):
    g = gen(4)
    ids = torch.randint(0, 6, (500,), generator=g, device="cuda", dtype=torch.int32)
    dout = rand(g, 500, 24)
    want, bound = ref.embedding_grad(dout, ids, 6, 1.0, 5)
    dout[ids == 5] = math.nan
    table = rand(g, 6, 24)
    table[5] = math.inf
    ref.within(ops.embedding_backward(dout, ids, 6, pad_id=5), want, bound)
    assert (ops.embedding(table, ids, pad_id=5)[ids == 5] == 0).all()


# ------------------------------------------------------------- layer norm
ROWS_WIDTHS = [(1, 1), (3, 2), (1, 256), (9, 31), (17, 32), (8, 33), (5, 100), (300, 128),
               (1000, 256), (33, 634), (7, 768), (10, 1023), (10, 1024), (4, 1025), (300, 1028),
               (5, 2050), (40, 5001), (160, 8192), (6000, 36), (5000, 61)]


@pytest.mark.parametrize("xd,yd", list(itertools.product([F32, BF16], repeat=2)))
@pytest.mark.parametrize("rows,width", ROWS_WIDTHS)
def test_layer_norm(ops, xd, yd, rows, width):
    g = gen(rows + width)
    x = (rand(g, rows, width) * (0.2 + 3 * torch.rand(rows, 1, generator=g, device="cuda"))
         + 5 * rand(g, rows, 1)).to(xd)
    gamma, beta = 1 + 0.3 * rand(g, width), rand(g, width)
    eps = float(torch.tensor(1e-5, dtype=F32))
    f = ref.norm(x, gamma, beta, eps)
    y, mean, rstd = ops.layer_norm(x, gamma, beta, out_dtype=yd)
    assert y.dtype == yd
    ref.within(y, f["y"], f["e_y"] + ref.HALF[yd] * (f["y"].abs() + f["e_y"]), "y")
    ref.within(mean, f["mean"][:, 0], f["e_mean"][:, 0], "mean")
    ref.within(rstd, f["rstd"][:, 0], f["e_rstd"][:, 0], "rstd")
    y2, none, _ = ops.layer_norm(x, gamma, beta, out_dtype=yd, stats=False)
    assert none is None and torch.equal(y, y2)
    dy = rand(g, rows, width, dtype=yd)
    for dres in (None, rand(g, rows, width, dtype=xd)):
        dx, e_dx, dg, e_dg, db, e_db = ref.norm_grad(f, dy, dres, xd)
        got = ops.layer_norm_backward(dy, x, gamma, mean, rstd, dres=dres)
        assert got[0].dtype == xd
        # the stored statistics the backward reads are the ones bounded above
        ref.within(got[0], dx, 2 * e_dx, "dx")
        ref.within(got[1], dg, 2 * e_dg, "dgamma")
        ref.within(got[2], db, e_db, "dbeta")
        again = ops.layer_norm_backward(dy, x, gamma, mean, rstd, dres=dres)
        assert all(torch.equal(a, b) for a, b in zip(got, again))
    base = rand(g, 2, width)
    acc = ops.layer_norm_backward(dy, x, gamma, mean, rstd, dgamma=base[0].clone(),
                                  dbeta=base[1].clone(), accumulate=True)
    ref.within(acc[1], base[0].double() + dg, 2 * e_dg + 2 * ref.U * (base[0].abs() + dg.abs()))
    ref.within(acc[2], base[1].double() + db, e_db + 2 * ref.U * (base[1].abs() + db.abs()))
    only = ops.layer_norm_backward(dy, x, gamma, mean, rstd, weight_grads=False)
    assert only[1] is None and only[2] is None
    ref.within(only[0], ref.norm_grad(f, dy, None, xd)[0], 2 * ref.norm_grad(f, dy, None, xd)[1], "dx alone")


def test_layer_norm_plain_views_and_empty(ops):
    g = gen(9)
    eps = float(torch.tensor(1e-5, dtype=F32))
    big = rand(g, 4, 6, 300)
    for x in (big, big[..., 20:120], big[..., 1:98], big[:, ::2], big.transpose(0, 1),
              big[:1].expand(4, 6, 300)):
        f = ref.norm(x, None, None, eps)
        y, mean, rstd = ops.layer_norm(x)
        ref.within(y, f["y"], f["e_y"] + ref.U * f["y"].abs())
        dy = rand(g, *x.shape)
        dx, e_dx, dg, e_dg, db, e_db = ref.norm_grad(f, dy, None, F32)
        got = ops.layer_norm_backward(dy, x, None, mean, rstd)
        ref.within(got[0], dx, 2 * e_dx)
        ref.within(got[1], dg, 2 * e_dg)
        ref.within(got[2], db, e_db)
    e = torch.zeros(0, 300, device="cuda")
    y, mean, rstd = ops.layer_norm(e)
    assert y.shape == (0, 300) and mean.shape == (0,)
    dx, dg, db = ops.layer_norm_backward(e, e, None, mean, rstd)
    assert dx.shape == (0, 300) and (dg == 0).all() and (db == 0).all()


@pytest.mark.parametrize("xd,yd", list(itertools.product([F32, BF16], repeat=2)))
@pytest.mark.parametrize("width", [3, 62, 127, 130, 509, 1021, 1023, 1026, 2051, 4099, 8191])
def test_layer_norm_row_phases(ops, xd, yd, width):
    """Rows that start anywhere: odd pitches, tensors that start off a boundary
    together or apart, rows enough for every block to take several."""
    g = gen(width)
    rows = 1300 if width < 1100 else 701
    eps = float(torch.tensor(1e-5, dtype=F32))
    gamma, beta = 1 + 0.3 * rand(g, width), rand(g, width)
    for pitch, offs in ((width, 0), (width + 2, 1), (width + 5, 3), (width + 8, 2)):
        buf = rand(g, rows * pitch + 8, dtype=xd)
        x = buf[offs:offs + rows * pitch].view(rows, pitch)[:, :width]
        f = ref.norm(x, gamma, beta, eps)
        y, mean, rstd = ops.layer_norm(x, gamma, beta, out_dtype=yd)
        ref.within(y, f["y"], f["e_y"] + ref.HALF[yd] * (f["y"].abs() + f["e_y"]), "y")
        gb = rand(g, rows * pitch + 8, dtype=yd)
        for o2 in (offs, (offs + 1) % 4):            # at x's phase, and at another
            dy = gb[o2:o2 + rows * pitch].view(rows, pitch)[:, :width]
            dx, e_dx, dg, e_dg, db, e_db = ref.norm_grad(f, dy, x, xd)
            got = ops.layer_norm_backward(dy, x, gamma, mean, rstd, dres=x)
            ref.within(got[0], dx, 2 * e_dx, "dx")
            ref.within(got[1], dg, 2 * e_dg, "dgamma")
            ref.within(got[2], db, e_db, "dbeta")


def test_layer_norm_in_place(pkg, ops):
    """y over x, dx over dres and dx over dy through the C entry."""
    import ptcg_b200.native as n
    lib, g = n.lib(), gen(11)
    s = torch.cuda.current_stream().cuda_stream
    for rows, width in ((37, 256), (21, 2600), (13, 77)):
        x = rand(g, rows, width)
        gamma, beta = rand(g, width), rand(g, width)
        y, mean, rstd = ops.layer_norm(x, gamma, beta)
        z = x.clone()
        p = lambda t: t.data_ptr()                                     # noqa: E731
        assert lib.ptcg_layer_norm_fwd(p(z), 0, width, p(gamma), p(beta), 1e-5, p(z), 0, width,
                                       None, None, rows, width, s) == 0
        assert torch.equal(z, y)
        dy, dres = rand(g, rows, width), rand(g, rows, width)
        dx, dg, db = ops.layer_norm_backward(dy, x, gamma, mean, rstd, dres=dres)
        need = lib.ptcg_layer_norm_bwd_scratch(rows, width)
        scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
        for over in (dres.clone(), dy.clone()):
            src = {"dy": dy, "dres": dres}
            src["dres" if torch.equal(over, dres) else "dy"] = over
            w = torch.empty(2, width, device="cuda")
            assert lib.ptcg_layer_norm_bwd(
                p(src["dy"]), 0, width, p(x), 0, width, p(gamma), p(mean), p(rstd), p(src["dres"]),
                width, p(over), width, p(w[0]), p(w[1]), 0, rows, width, p(scratch), need, s) == 0
            assert torch.equal(over, dx) and torch.equal(w[0], dg) and torch.equal(w[1], db)


def test_layer_norm_constant_and_far_rows(ops):
    """A constant row has variance 0 (y = beta); a row far from 0 keeps its
    digits, since the variance is taken about the mean."""
    x = torch.full((3, 640), 12345.0, device="cuda")
    y, mean, rstd = ops.layer_norm(x, None, torch.full((640,), 0.5, device="cuda"))
    assert (mean == 12345).all() and (y == 0.5).all()
    eps = float(torch.tensor(1e-5, dtype=F32))
    assert torch.allclose(rstd.double(), torch.full((3,), eps ** -0.5, device="cuda", dtype=torch.float64),
                          rtol=2 ** -20)


@pytest.mark.parametrize("xd,at", [(F32, 12345.0), (F32, -0.1), (BF16, 12352.0)])
@pytest.mark.parametrize("width", [1, 3, 56, 60, 112, 120, 224, 240, 252, 380, 639, 1000, 1028, 2051, 5001, 8191])
def test_layer_norm_constant_rows_of_any_width(ops, xd, at, width):
    """Whatever the width's reciprocal rounds to: the mean is the value, the
    deviations are 0."""
    x = torch.full((5, width), at, device="cuda", dtype=xd)
    y, mean, rstd = ops.layer_norm(x, None, torch.full((width,), 0.5, device="cuda"))
    assert (mean == x[:, 0].float()).all() and (y == 0.5).all()
    eps = float(torch.tensor(1e-5, dtype=F32))
    assert ((rstd.double() / eps ** -0.5 - 1).abs() <= ref.FN).all()


@pytest.mark.parametrize("width", [1, 3, 56, 60, 120, 240, 380, 639, 1000, 1028, 2051, 5001, 8191])
def test_layer_norm_far_rows_with_variance(ops, width):
    """Rows some 10^4 from 0 whose deviations are a few steps of fp32 there: y
    is as exact as the deviations' own arithmetic.  c = x - mean, e the first
    pass's mean's error (a step per addition): x - mu is exact, its sum is off
    by depth u of its terms' magnitudes, at most |c| + e, and the variance
    about it likewise; the first-order error of the mean does not appear."""
    g = gen(width)
    rows = 9
    x = 1e4 + 0.01 * rand(g, rows, width) * (1 + 10 * torch.rand(rows, 1, generator=g, device="cuda"))
    gamma, beta = 1 + 0.3 * rand(g, width), rand(g, width)
    eps = float(torch.tensor(1e-5, dtype=F32))
    f = ref.norm(x, gamma, beta, eps)
    c = f["x"] - f["mean"]
    off = f["e_mean"]
    size = c.abs().mean(-1, keepdim=True) + off
    e_dm = (f["depth"] + 3) * ref.U * size
    e_var = (f["depth"] + 8) * ref.U * ((c.abs() + off) ** 2).mean(-1, keepdim=True)
    rel_r = 0.5 * e_var / ((c * c).mean(-1, keepdim=True) + eps) + ref.FN
    e_h = f["rstd"] * e_dm + f["h"].abs() * (rel_r + 3 * ref.U)
    e_y = f["g"].abs() * e_h + 3 * ref.U * ((f["h"] * f["g"]).abs() + beta.double().abs())
    y, mean, rstd = ops.layer_norm(x, gamma, beta)
    ref.within(y, f["y"], e_y, "y")
    ref.within(mean, f["mean"][:, 0], (e_dm + ref.U * f["mean"].abs())[:, 0], "mean")
    ref.within(rstd, f["rstd"][:, 0], (f["rstd"] * rel_r)[:, 0], "rstd")


@pytest.mark.parametrize("width", [1, 37, 62, 100, 127, 130])
@pytest.mark.parametrize("at", [3e19, -2e36])
def test_layer_norm_huge_constant_rows(ops, at, width):
    """One last place of the mean, squared, is past fp32's range there; the
    variance is 0 all the same."""
    x = torch.full((5, width), at, device="cuda")
    y, mean, rstd = ops.layer_norm(x)
    assert (y == 0).all() and (mean == x[:, 0]).all()
    eps = float(torch.tensor(1e-5, dtype=F32))
    assert ((rstd.double() / eps ** -0.5 - 1).abs() <= ref.FN).all()


@pytest.mark.parametrize("xd,yd", list(itertools.product([F32, BF16], repeat=2)))
@pytest.mark.parametrize("rows,width", [(1, 3), (70001, 64), (70001, 5), (6001, 1024), (40000, 255), (5003, 2050),
                                        (3001, 5001), (2000, 8192)])
def test_layer_norm_weight_gradients_exact_sums(ops, xd, yd, rows, width):
    """Whole numbers of -3 to 3 with mean 0 and rstd 1 given, so that h = x and
    all sums stay below 2^24: exact in any order, and no row may be missing."""
    g = gen(rows)
    x, dy = (torch.randint(-3, 4, (rows, width), generator=g, device="cuda").to(t) for t in (xd, yd))
    mean, rstd = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    _, dg, db = ops.layer_norm_backward(dy, x, None, mean, rstd)
    assert 9 * rows < 2 ** 24
    assert torch.equal(dg.double(), (dy.double() * x.double()).sum(0))
    assert torch.equal(db.double(), dy.double().sum(0))


@pytest.mark.parametrize("width,pitch,offset", [(37, 37, 0), (100, 100, 0), (37, 39, 1), (62, 62, 2), (130, 130, 0)])
def test_layer_norm_gradient_of_huge_rows(ops, width, pitch, offset):
    """Constant rows so large that mean * rstd is past fp32's range: h is 0, and
    dx is the gradient less its mean, times rstd."""
    buf = torch.full((3 * pitch + 4,), 2e36, device="cuda")
    x = buf[offset:offset + 3 * pitch].view(3, pitch)[:, :width]
    y, mean, rstd = ops.layer_norm(x)
    assert (y == 0).all()
    dy = rand(gen(width), 3 * pitch + 4)[offset:offset + 3 * pitch].view(3, pitch)[:, :width]
    f = ref.norm(torch.zeros(3, width, device="cuda"), None, None, float(torch.tensor(1e-5, dtype=F32)))
    dx, e_dx, dg, e_dg, db, e_db = ref.norm_grad(f, dy, None, F32)
    got = ops.layer_norm_backward(dy, x, None, mean, rstd)
    ref.within(got[0], dx, 2 * e_dx, "dx")
    assert (got[1] == 0).all()
    ref.within(got[2], db, e_db, "dbeta")


# -------------------------------------------------------- cross attention
def problem(seed, nseq, lq, lk, heads, kvh, dh, dtype, mask, layout="rows"):
    g = gen(seed)
    q = rand(g, nseq, lq, heads, dh, dtype=dtype)
    if layout == "heads":
        k, v = (rand(g, nseq, kvh, lk, dh, dtype=dtype).transpose(1, 2) for _ in range(2))
    elif layout == "packed":                     # q as a slice, k and v interleaved
        q = rand(g, nseq, lq, heads, 3 * dh, dtype=dtype)[..., dh:2 * dh]
        k, v = rand(g, nseq, lk, 2, kvh, dh, dtype=dtype).unbind(2)
    else:
        k, v = (rand(g, nseq, lk, kvh, dh, dtype=dtype) for _ in range(2))
    keep = kv_len = None
    if "keep" in mask:
        keep = torch.rand(nseq, lk, generator=g, device="cuda") < 0.6
        keep[nseq // 2] = False                  # a sequence without a key
        keep[0, : lk // 2] = False               # leading holes, tiles with no key
    if "len" in mask:
        kv_len = torch.randint(-2, lk + 4, (nseq,), generator=g, device="cuda", dtype=torch.int32)
        kv_len[0], kv_len[-1] = lk, 0
    return q, k, v, {"keep": keep, "kv_len": kv_len}


def run_cross(ops, q, k, v, mask, scale=None, seed=5):
    dout = rand(gen(seed), *q.shape, dtype=q.dtype)
    out, lse = ops.cross_attention(q, k, v, scale=scale, **mask)
    grads = ops.cross_attention_backward(dout, q, k, v, out, lse, scale=scale, **mask)
    return dout, (out, lse, *grads)


def check_cross(ops, q, k, v, mask, scale=None):
    dout, got = run_cross(ops, q, k, v, mask, scale)
    r = ref.cross(q, k, v, scale=scale, dout=dout, **mask)
    for name, t in zip(("out", "lse", "dq", "dk", "dv"), got):
        assert t.dtype == (F32 if name == "lse" else q.dtype)
        ref.within(t, r[name], r["e_" + name], name)
    live = ref.live_keys(k.shape[0], k.shape[1], mask["keep"], mask["kv_len"], "cuda")
    assert (got[3][~live] == 0).all() and (got[4][~live] == 0).all()
    empty = ~live.any(-1)
    assert (got[0][empty] == 0).all() and (got[2][empty] == 0).all()
    assert (got[1][empty] == -math.inf).all()
    return dout, got


CROSS = [  # nseq, lq, lk, heads, kv_heads, dh
    (1, 1, 1, 1, 1, 32), (4, 1, 129, 8, 8, 32), (3, 1, 700, 8, 2, 64), (2, 1, 3000, 8, 1, 128),
    (5, 64, 129, 8, 8, 32), (3, 17, 63, 4, 2, 64), (2, 65, 64, 2, 2, 128), (2, 130, 65, 4, 1, 32),
    (1, 63, 1000, 2, 1, 128), (1, 700, 33, 3, 3, 64), (1, 1500, 70, 2, 1, 32), (7, 5, 8, 6, 3, 32),
    (2, 16, 257, 1, 1, 128), (1, 300, 520, 4, 4, 128), (300, 9, 31, 2, 1, 32), (4, 31, 150, 2, 2, 128),
    (3, 10, 70, 4, 2, 64), (2, 24, 2100, 2, 2, 32)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("mask", ["none", "keep", "len", "keep len"])
@pytest.mark.parametrize("nseq,lq,lk,heads,kvh,dh", CROSS)
def test_cross_attention(ops, dtype, mask, nseq, lq, lk, heads, kvh, dh):
    q, k, v, m = problem(nseq * lq + lk, nseq, lq, lk, heads, kvh, dh, dtype, mask)
    dout, got = check_cross(ops, q, k, v, m)
    again = run_cross(ops, q, k, v, m)[1]
    assert all(torch.equal(a, b) for a, b in zip(got, again))


LONG = [  # the shapes of the long-problem kernels: nseq, lq, lk, heads, kv_heads, dh
    (1, 65, 129, 1, 1, 64), (1, 128, 256, 2, 2, 128), (2, 300, 520, 2, 1, 128), (2, 400, 300, 2, 2, 32),
    (1, 1100, 700, 2, 1, 64), (3, 70, 2000, 2, 2, 128), (2, 129, 385, 3, 1, 32), (1, 1500, 1025, 1, 1, 32),
    (40, 80, 100, 4, 4, 64), (1, 257, 65, 1, 1, 128)]


@pytest.mark.parametrize("mask", ["none", "keep", "len", "keep len"])
@pytest.mark.parametrize("layout", ["rows", "heads", "packed"])
@pytest.mark.parametrize("nseq,lq,lk,heads,kvh,dh", LONG)
def test_cross_attention_long(pkg, ops, mask, layout, nseq, lq, lk, heads, kvh, dh):
    import ptcg_b200.native as n
    q, k, v, m = problem(lq + lk, nseq, lq, lk, heads, kvh, dh, BF16, mask, layout)
    dout, got = check_cross(ops, q, k, v, m)
    assert n.lib().ptcg_device_error() == 0
    for _ in range(3):
        again = run_cross(ops, q, k, v, m)[1]
        assert all(torch.equal(a, b) for a, b in zip(got, again))
    live = ref.live_keys(nseq, lk, m["keep"], m["kv_len"], "cuda")
    if not live.all():                              # masked rows may hold anything
        kj, vj = k.clone(), v.clone()
        kj[~live] = math.nan
        vj[~live] = math.nan
        assert all(torch.equal(a, b) for a, b in zip(run_cross(ops, q, kj, vj, m)[1], got))
    # one encoder's states for every sequence, and one key head's for all heads
    check_cross(ops, q, k[:1].expand_as(k), v[:1].expand_as(v), m)
    check_cross(ops, q, k[:, :, :1].expand_as(k), v[:, :, :1].expand_as(v), m)


def test_cross_attention_long_growing_scores(ops):
    """Maxima that rise by small and large steps along the keys: the shift of
    a row lags behind its maximum by up to 2^8, then its output is rescaled."""
    for dh in (32, 64, 128):
        for top in (2.0, 14.0):
            q, k, v, m = problem(29, 1, 400, 900, 1, 1, dh, BF16, "none")
            k = k * torch.linspace(0.1, top, 900, device="cuda", dtype=BF16).view(1, 900, 1, 1)
            check_cross(ops, q * 2, k, v, m)
            check_cross(ops, q * 2, k.flip(1), v, m)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens", ["drawn", "none", "one", "equal", "short"])
@pytest.mark.parametrize("nseq,lq,lk,heads,kvh,dh", [(5, 1, 9000, 8, 2, 64), (40, 2, 4100, 2, 1, 32),
                                                     (3, 4, 20000, 4, 1, 128), (1, 1, 4096, 3, 3, 128),
                                                     (147, 1, 4200, 2, 2, 32)])
def test_cross_attention_uneven_caches(ops, dtype, lens, nseq, lq, lk, heads, kvh, dh):
    """Single tokens over long caches of unequal lengths, which the blocks share
    out by the lengths: empty caches, one that has all keys, few keys in all."""
    q, k, v, _ = problem(lk, nseq, lq, lk, heads, kvh, dh, dtype, "none", "rows")
    n = torch.randint(0, lk + 1, (nseq,), generator=torch.Generator().manual_seed(nseq), dtype=torch.int32)
    if lens == "none":
        n[:] = 0
    elif lens == "one":
        n[:] = 0
        n[nseq // 2] = lk
    elif lens == "equal":
        n[:] = lk
    elif lens == "short":
        n %= 70
    m = {"keep": None, "kv_len": n.cuda()}
    out, lse = ops.cross_attention(q, k, v, **m)
    r = ref.cross(q, k, v, **m)
    ref.within(out, r["out"], r["e_out"], "out")
    ref.within(lse, r["lse"], r["e_lse"], "lse")
    again, _ = ops.cross_attention(q, k, v, **m)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["heads", "packed"])
@pytest.mark.parametrize("nseq,lq,lk,heads,kvh,dh", [(3, 40, 75, 4, 2, 32), (2, 1, 900, 4, 4, 64),
                                                     (2, 90, 40, 2, 2, 128)])
def test_cross_attention_layouts(ops, dtype, layout, nseq, lq, lk, heads, kvh, dh):
    q, k, v, m = problem(7, nseq, lq, lk, heads, kvh, dh, dtype, "keep len", layout)
    check_cross(ops, q, k, v, m, scale=0.37)
    # one encoder's states for every sequence: their gradients come per sequence
    check_cross(ops, q, k[:1].expand_as(k), v[:1].expand_as(v), m)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lq", [1, 40])
def test_cross_attention_masked_keys_may_hold_anything(ops, dtype, lq):
    q, k, v, m = problem(13, 4, lq, 600, 4, 2, 64, dtype, "keep len")
    dout, want = run_cross(ops, q, k, v, m)
    live = ref.live_keys(4, 600, m["keep"], m["kv_len"], "cuda")
    for junk in (math.nan, math.inf, -math.inf, torch.finfo(dtype).min):
        kj, vj = k.clone(), v.clone()
        kj[~live] = junk
        vj[~live] = junk
        got = run_cross(ops, q, kj, vj, m)[1]
        assert all(torch.equal(a, b) for a, b in zip(got, want)), junk
    # keep as bytes other than 0 / 1
    m8 = {"keep": m["keep"].to(torch.uint8) * 255, "kv_len": m["kv_len"]}
    assert all(torch.equal(a, b) for a, b in zip(run_cross(ops, q, k, v, m8)[1], want))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nseq,lq,lk,dh", [(2, 20, 50, 64), (2, 20, 600, 64), (2, 100, 50, 64), (2, 100, 200, 128),
                                           (1, 3000, 60, 32), (2, 600, 700, 64), (1, 7, 3000, 32)])
def test_cross_attention_masked_keys_take_no_gradient(ops, dtype, nseq, lq, lk, dh):
    """Nor where dout holds infinities or NaN: 0 times those is not 0."""
    q, k, v, m = problem(lq, nseq, lq, lk, 4, 2, dh, dtype, "keep len")
    live = ref.live_keys(nseq, lk, m["keep"], m["kv_len"], "cuda")
    if nseq == 1:                                # problem() empties the only one
        m["keep"][:] = torch.rand(1, lk, generator=gen(3), device="cuda") < 0.6
        m["kv_len"][:] = lk - 7
        live = ref.live_keys(nseq, lk, m["keep"], m["kv_len"], "cuda")
    dout = rand(gen(5), *q.shape, dtype=dtype)
    dout[0, lq // 2, 1, 5], dout[0, lq - 1, 3, dh - 1] = math.inf, math.nan
    out, lse = ops.cross_attention(q, k, v, **m)
    dq, dk, dv = ops.cross_attention_backward(dout, q, k, v, out, lse, **m)
    assert live.any() and not live.all()
    assert (dk[~live] == 0).all() and (dv[~live] == 0).all()
    assert not dv[live].isfinite().all()         # a kept key does take them


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_cross_attention_no_lengths(ops, dtype):
    z = lambda *s: torch.zeros(*s, device="cuda", dtype=dtype)     # noqa: E731
    out, lse = ops.cross_attention(z(2, 3, 4, 32), z(2, 0, 2, 32), z(2, 0, 2, 32))
    assert (out == 0).all() and (lse == -math.inf).all()
    dq, dk, dv = ops.cross_attention_backward(out, z(2, 3, 4, 32), z(2, 0, 2, 32), z(2, 0, 2, 32), out, lse)
    assert (dq == 0).all() and dk.shape == (2, 0, 2, 32)
    q, k = z(2, 0, 4, 32), z(2, 70, 2, 32) + 1
    out, lse = ops.cross_attention(q, k, k)
    assert out.shape == (2, 0, 4, 32) and lse.shape == (2, 4, 0)
    dq, dk, dv = ops.cross_attention_backward(out, q, k, k, out, lse)
    assert (dk == 0).all() and (dv == 0).all()
    out, lse = ops.cross_attention(z(0, 3, 4, 32), z(0, 70, 2, 32), z(0, 70, 2, 32))
    assert out.shape == (0, 3, 4, 32)


def test_cross_attention_long_sums(ops):
    """fp32 sums over many keys or rows are as exact as short ones."""
    for nseq, lq, lk, heads, kvh, dh in ((1, 48, 20000, 2, 2, 32), (1, 100, 20000, 2, 1, 128), (1, 6000, 100, 1, 1, 64)):
        q, k, v, m = problem(lk, nseq, lq, lk, heads, kvh, dh, F32, "none", "rows")
        dout, got = run_cross(ops, q, k, v, m)
        r = ref.cross(q, k, v, dout=dout, **m)
        for name, t in zip(("out", "dq", "dk", "dv"), (got[0], got[2], got[3], got[4])):
            err = float((t.double() - r[name]).pow(2).mean().sqrt() / r[name].pow(2).mean().sqrt())
            # P = exp(s - lse): s of some 4 and lse of some 10 are off by half a
            # step each, 2^-22 + 2^-21, the products and sums by less; in the root
            # mean square below that, so 2^-20 holds with room
            assert err < 2.0 ** -20, (name, err)


@pytest.mark.parametrize("lq", [1, 20, 40, 100])
def test_cross_attention_small_probabilities(ops, lq):
    """fp32 probabilities down to e^-82 are as exact as large ones.  The scores
    are whole numbers, so they are exact; one is 0 and the rest below e^-20, so
    that the sum rounds to 1 and the log-sum-exp to 0 (both true to 2^-28).  Each
    result that is looked at is one exponential, off by 2 units of the last
    place (4 u), times factors that are exact or off by a few u: out 3 P (u each
    from the division and the product), dv P, dq P (dP - delta) with dP = 3 and
    delta = 1 (2 u of it, which is u of the difference of 2, and u each from
    the difference, the product and the last factor)."""
    dh = 32
    z = lambda n: torch.zeros(1, n, 1, dh, device="cuda")          # noqa: E731
    q, k, v, dout = z(lq), z(dh), z(dh), z(lq)
    s = torch.tensor([0.0] + [-20.0 - 2 * j for j in range(1, dh)], device="cuda")
    q[..., 0] = 1
    k[0, :, 0, 0] = s
    v[0, 0, 0, 0] = 1
    for j in range(1, dh):
        k[0, j, 0, j], v[0, j, 0, j] = 1, 3
    out, lse = ops.cross_attention(q, k, v, scale=1.0)
    p = torch.softmax(s.double(), 0)
    off = lambda got, want: ((got.double() / want - 1).abs().max() / ref.U).item()   # noqa: E731
    assert (lse == 0).all()
    assert off(out[0, :, 0, 1:], 3 * p[1:]) <= 7
    dout[0, lq - 1] = 1
    dq, dk, dv = ops.cross_attention_backward(dout, q, k, v, out, lse, scale=1.0)
    assert off(dv[0, :, 0], p[:, None].expand(dh, dh)) <= 7
    assert off(dq[0, lq - 1, 0, 1:], 2 * p[1:]) <= 9


@pytest.mark.parametrize("even", [False, True])
@pytest.mark.parametrize("lq", [1, 20, 100])
def test_cross_attention_parts_of_large_scores(ops, even, lq):
    """fp32 keys that are split into parts and joined keep what scores of 1000
    have left: eight scores that are exact, one in every eighth of the cache.
    Per column one part counts: its weight is one exponential (4 u, the
    difference in it exact), over the sum of eight (4 u, and u for each of seven
    additions in some order), and u each for the reciprocal and the product;
    where parts hold several of the keys their own sums and factors come to
    another 12 u at most."""
    dh, lk, n = 32, 8192, 8
    q, k, v = (torch.zeros(1, r, 1, dh, device="cuda") for r in (lq, lk, lk))
    keep = torch.zeros(1, lk, dtype=torch.bool, device="cuda")
    s = torch.tensor([1000 - 1.375 * ((3 * b) % n) for b in range(n)], device="cuda")
    q[..., 0] = 1
    for b in range(n):
        at = b * (lk // n) + 5
        keep[0, at], k[0, at, 0, 0], v[0, at, 0, b] = True, s[b], 1
    kv_len = torch.tensor([lk], dtype=torch.int32, device="cuda") if even else None
    out, lse = ops.cross_attention(q, k, v, keep=keep, kv_len=kv_len, scale=1.0)
    p = torch.softmax(s.double(), 0)
    assert ((out[..., :n].double() / p - 1).abs() <= 29 * ref.U).all()
    want = torch.logsumexp(s.double(), 0)
    assert ((lse.double() - want).abs() <= ref.U * want + 16 * ref.U).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_cross_attention_large_scores(ops, dtype):
    """Scores of hundreds: the running maximum keeps every exponential in
    range, and rows whose maximum comes last are rescaled."""
    q, k, v, m = problem(17, 2, 33, 300, 2, 2, 32, dtype, "none")
    k = k * torch.linspace(0.1, 12, 300, device="cuda", dtype=dtype).view(1, 300, 1, 1)
    q = q * 4
    check_cross(ops, q, k, v, m)
    check_cross(ops, q, k.flip(1), v, m)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_cross_attention_offsets_past_32_bits(ops, dtype):
    """Sequences of one cache that lie more than 2^31 elements apart."""
    far = (1 << 31) + 64
    buf = torch.empty(far + 70 * 2 * 64, device="cuda", dtype=dtype)
    k = buf.as_strided((2, 70, 2, 32), (far, 128, 32, 1))
    v = buf.as_strided((2, 70, 2, 32), (far, 128, 32, 1), 64)
    q, k0, v0, m = problem(19, 2, 21, 70, 4, 2, 32, dtype, "none")
    k.copy_(k0)
    v.copy_(v0)
    check_cross(ops, q, k, v, m)


def test_cross_attention_gradient_against_differences(ops):
    """The fp32 gradients along a direction against central differences of the
    formula in 64 bits (step 1e-5: the difference itself is good to 1e-9 of
    the sums involved, below the gradient's own bound)."""
    q, k, v, m = problem(23, 3, 19, 45, 4, 2, 32, F32, "keep len")
    dout, got = run_cross(ops, q, k, v, m)
    r = ref.cross(q, k, v, dout=dout, **m)
    loss = lambda a, b, c: (ref.cross(a, b, c, **m)["out"] * dout.double()).sum()   # noqa: E731
    base = [t.double() for t in (q, k, v)]
    for i, name in enumerate(("dq", "dk", "dv")):
        d = rand(gen(i), *base[i].shape).double()
        plus, minus = list(base), list(base)
        plus[i], minus[i] = base[i] + 1e-5 * d, base[i] - 1e-5 * d
        diff = (loss(*plus) - loss(*minus)) / 2e-5
        along = (got[2 + i].double() * d).sum()
        bound = (r["e_" + name] * d.abs()).sum() + 1e-8 * (r[name] * d).abs().sum()
        assert (diff - along).abs() <= bound, name


# ------------------------------------------------------------ all together
def decoder(ops, w, ids, enc, mask, dy=None):
    """One pre-norm decoder sublayer: embedded options, norm, cross attention
    to the encoder's rows, residual; with dy also the gradients of the table,
    the norm and the encoder's keys and values."""
    n, lq = ids.shape
    x = ops.embedding(w["table"], ids, scale=2.0, pad_id=0)
    h, mean, rstd = ops.layer_norm(x, w["gamma"], w["beta"], out_dtype=BF16)
    q = h.view(n, lq, 4, 32)
    k, v = enc[..., :64].unflatten(-1, (2, 32)), enc[..., 64:].unflatten(-1, (2, 32))
    out, lse = ops.cross_attention(q, k, v, **mask)
    y = x + out.reshape(n, lq, 128).float()
    if dy is None:
        return (y,)
    dq, dk, dv = ops.cross_attention_backward(dy.to(BF16).view_as(q), q, k, v, out, lse, **mask)
    dx, dg, db = ops.layer_norm_backward(dq.view(n, lq, 128), x, w["gamma"], mean, rstd, dres=dy)
    return y, ops.embedding_backward(dx, ids, w["table"].shape[0], scale=2.0, pad_id=0), dg, db, dk, dv


def decoder_inputs(seed):
    g = gen(seed)
    w = {"table": rand(g, 50, 128), "gamma": 1 + 0.1 * rand(g, 128), "beta": 0.1 * rand(g, 128)}
    ids = torch.randint(0, 50, (6, 13), generator=g, device="cuda", dtype=torch.int32)
    enc = rand(g, 6, 37, 128, dtype=BF16)
    keep = torch.rand(6, 37, generator=g, device="cuda") < 0.7
    return w, ids, enc, {"keep": keep, "kv_len": None}, rand(g, 6, 13, 128)


def test_decoder_sublayer_against_autograd(ops):
    """The chain against 64-bit autograd of the same formulas.  Every value
    passes two or three bf16 roundings (2^-8 each: h, out, dq and the operands
    P and dS), so each result is within 4 * 2^-8 in 2-norm."""
    w, ids, enc, mask, dy = decoder_inputs(31)
    got = decoder(ops, w, ids, enc, mask, dy)
    t, ga, be, en = (a.double().requires_grad_() for a in (w["table"], w["gamma"], w["beta"], enc))
    x = t[ids.long()] * 2.0 * (ids != 0)[..., None]
    h = torch.nn.functional.layer_norm(x, (128,), ga, be)
    q = h.view(6, 13, 4, 32)
    k, v = (en[..., i:i + 64].unflatten(-1, (2, 32)).repeat_interleave(2, 2) for i in (0, 64))
    s = torch.einsum("nihd,njhd->nhij", q, k) / math.sqrt(32)
    p = torch.softmax(s.masked_fill(~mask["keep"][:, None, None, :], -math.inf), -1)
    y = x + torch.einsum("nhij,njhd->nihd", p, v).reshape(6, 13, 128)
    y.backward(dy.double())
    want = (y, t.grad, ga.grad, be.grad, en.grad[..., :64].unflatten(-1, (2, 32)),
            en.grad[..., 64:].unflatten(-1, (2, 32)))
    for i, (a, b) in enumerate(zip(got, want)):
        assert (a.double() - b).norm() <= 4 * 2.0 ** -8 * b.norm(), i


def test_graph_replay_with_other_lengths(ops):
    """A captured single-token call shares its keys out by the lengths that are
    there when it is replayed."""
    q, k, v, _ = problem(4, 6, 1, 7000, 4, 2, 64, BF16, "none", "heads")
    n = torch.tensor([7000, 3, 0, 512, 4097, 6999], dtype=torch.int32, device="cuda")
    ops.cross_attention(q, k, v, kv_len=n)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out, lse = ops.cross_attention(q, k, v, kv_len=n)
    for lens in ([1, 1, 1, 1, 1, 1], [0, 7000, 0, 0, 0, 0], [9000, 255, 256, 257, -5, 6000]):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        gr.replay()
        want, wlse = ops.cross_attention(q, k, v, kv_len=n)
        assert torch.equal(out, want) and torch.equal(lse, wlse)
        r = ref.cross(q, k, v, kv_len=n)
        ref.within(out, r["out"], r["e_out"], "out")


def test_graph_capture_and_replay(ops):
    """Two captured graphs, replayed in turn on new inputs beside eager calls,
    give the eager results bit for bit."""
    sets = [decoder_inputs(s) for s in (41, 42)]
    eager = [decoder(ops, *s) for s in sets]
    graphs = []
    for _ in range(2):
        w, ids, enc, mask, dy = decoder_inputs(43)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            decoder(ops, w, ids, enc, mask, dy)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = decoder(ops, w, ids, enc, mask, dy)
        graphs.append((gr, (w, ids, enc, mask, dy), outs))
    for turn in range(4):
        gr, (w, ids, enc, mask, dy), outs = graphs[turn % 2]
        nw, nids, nenc, nmask, ndy = sets[turn // 2]
        for k in w:
            w[k].copy_(nw[k])
        ids.copy_(nids), enc.copy_(nenc), mask["keep"].copy_(nmask["keep"]), dy.copy_(ndy)
        gr.replay()
        beside = decoder(ops, *sets[turn // 2])
        torch.cuda.synchronize()
        for a, b, c in zip(outs, eager[turn // 2], beside):
            assert torch.equal(a, b) and torch.equal(c, b)


def test_two_streams_at_once(ops):
    """Calls that overlap on two streams share nothing."""
    sets = [decoder_inputs(s) for s in (51, 52)]
    want = [decoder(ops, *s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(decoder(ops, *sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def large_inputs(seed):
    """Problems whose kernels have something to collide over: tcgen05 with all
    of TMEM and split axes, single tokens in parts, a sort of several tiles."""
    g = gen(seed)
    q, k, v, _ = problem(seed, 1, 400, 2100, 2, 1, 128, BF16, "none")
    q1, k1, v1, _ = problem(seed + 1, 3, 1, 9000, 8, 2, 64, BF16, "none")
    n = torch.randint(0, 9001, (3,), generator=g, device="cuda", dtype=torch.int32)
    ids = torch.randint(0, 700, (20000,), generator=g, device="cuda", dtype=torch.int32)
    return [q, k, v, rand(g, *q.shape, dtype=BF16), q1, k1, v1, n, ids, rand(g, 20000, 48, dtype=BF16)]


def large_calls(ops, q, k, v, dout, q1, k1, v1, n, ids, demb):
    out, lse = ops.cross_attention(q, k, v)
    grads = ops.cross_attention_backward(dout, q, k, v, out, lse)
    return (out, lse, *grads, *ops.cross_attention(q1, k1, v1, kv_len=n),
            ops.embedding_backward(demb, ids, 700))


def test_two_streams_at_once_large(pkg, ops):
    """Large calls that overlap on two streams share nothing."""
    import ptcg_b200.native as n
    sets = [large_inputs(s) for s in (81, 91)]
    want = [large_calls(ops, *s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(large_calls(ops, *sets[i]))
    torch.cuda.synchronize()
    assert n.lib().ptcg_device_error() == 0
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_two_graphs_at_once_large(pkg, ops):
    """Two captured graphs of large calls, replayed on two streams at the same
    time, on inputs that were not there at the capture."""
    import ptcg_b200.native as n
    sets = [large_inputs(s) for s in (101, 111)]
    want = [large_calls(ops, *s) for s in sets]
    graphs = []
    for _ in range(2):
        inputs = large_inputs(121)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            large_calls(ops, *inputs)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = large_calls(ops, *inputs)
        graphs.append((gr, inputs, outs, side))
    for turn in range(4):
        for i, (gr, inputs, outs, side) in enumerate(graphs):
            for a, b in zip(inputs, sets[(i + turn) % 2]):
                a.copy_(b)
        torch.cuda.synchronize()
        for gr, _, _, side in graphs:
            with torch.cuda.stream(side):
                gr.replay()
        torch.cuda.synchronize()
        assert n.lib().ptcg_device_error() == 0
        for i, (gr, inputs, outs, side) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(outs, want[(i + turn) % 2]))


def test_under_an_autograd_function(ops):
    """The calls as the two passes of a Function: its leaves get the gradients
    that the calls return."""
    class Norm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, gamma, beta):
            y, mean, rstd = ops.layer_norm(x, gamma, beta)
            ctx.save_for_backward(x, gamma, mean, rstd)
            return y

        @staticmethod
        def backward(ctx, dy):
            return ops.layer_norm_backward(dy, *ctx.saved_tensors)

    g = gen(71)
    leaves = [t.requires_grad_() for t in (rand(g, 40, 96), rand(g, 96), rand(g, 96))]
    dy = rand(g, 40, 96)
    y = Norm.apply(*leaves)
    y.backward(dy)
    with torch.no_grad():
        y2, mean, rstd = ops.layer_norm(*leaves)
        want = ops.layer_norm_backward(dy, leaves[0], leaves[1], mean, rstd)
    assert torch.equal(y, y2) and all(torch.equal(t.grad, w) for t, w in zip(leaves, want))


def test_launches_are_counted(pkg, ops):
    import ptcg_b200.native as n
    lib = n.lib()
    before = lib.ptcg_launch_count()
    decoder(ops, *decoder_inputs(61))
    assert lib.ptcg_launch_count() - before >= 6         # one per call at least
