"""Refusals of the decoder operators, on the CPU: every bad argument is an
error code with a message before anything is launched, and the torch-facing
calls refuse mismatched tensors.  (Nothing here reaches a GPU.)"""
import ctypes as C

import pytest
import torch

OK, EINVAL, ERANGE = 0, 1, 4
BUF = (C.c_byte * 4096)()
A = (C.addressof(BUF) + 255) // 256 * 256          # a 256-byte aligned address


@pytest.fixture(scope="module")
def lib(pkg):
    import ptcg_b200.native as n
    return n.lib()


def emb_fwd(lib, table=A, td=0, ldt=8, vocab=4, width=8, ids=A, n=2, pad=-1, out=A, od=0, ldo=8):
    return lib.ptcg_embedding_fwd(table, td, ldt, vocab, width, ids, n, 1.0, pad, out, od, ldo, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(td=2), b"dtype"), (dict(od=-1), b"dtype"), (dict(vocab=0), b"bad sizes"),
    (dict(width=0), b"bad sizes"), (dict(n=-1), b"bad sizes"), (dict(ldt=7), b"bad sizes"),
    (dict(ldo=7), b"bad sizes"), (dict(table=None), b"null"), (dict(ids=None), b"null"),
    (dict(out=None), b"null"), (dict(table=A + 2), b"aligned"), (dict(ids=A + 1), b"aligned")])
def test_embedding_forward_refuses(lib, kw, msg):
    assert emb_fwd(lib, **kw) == EINVAL
    assert msg in lib.ptcg_last_error()


def emb_bwd(lib, dout=A, dd=0, lddo=8, ids=A, n=2, dtable=A, lddt=8, vocab=4, width=8, scratch=A,
            nbytes=1 << 30):
    return lib.ptcg_embedding_bwd(dout, dd, lddo, ids, n, 1.0, -1, dtable, lddt, vocab, width, 0,
                                  scratch, nbytes, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(dd=3), EINVAL), (dict(vocab=-1), EINVAL), (dict(width=0), EINVAL), (dict(n=-1), EINVAL),
    (dict(n=1 << 31), EINVAL), (dict(width=65535 * 32 + 1, lddo=1 << 22, lddt=1 << 22), EINVAL), (dict(lddo=4), EINVAL), (dict(lddt=4), EINVAL),
    (dict(dtable=None), EINVAL), (dict(dout=None), EINVAL), (dict(ids=None), EINVAL),
    (dict(scratch=None), EINVAL), (dict(scratch=A + 4), EINVAL), (dict(dtable=A + 2), EINVAL),
    (dict(nbytes=16), ERANGE)])
def test_embedding_gradient_refuses(lib, kw, rc):
    assert emb_bwd(lib, **kw) == rc
    assert b"embedding gradient" in lib.ptcg_last_error()


def test_embedding_scratch_size(lib):
    assert lib.ptcg_embedding_bwd_scratch(0, 10, 8) == 0
    assert lib.ptcg_embedding_bwd_scratch(-1, 10, 8) == -1
    assert lib.ptcg_embedding_bwd_scratch(1 << 31, 10, 8) == -1
    assert lib.ptcg_embedding_bwd_scratch(5, 0, 8) == -1
    assert lib.ptcg_embedding_bwd_scratch(5, 8, 65535 * 32 + 1) == -1
    # two sets of keys and places at least
    assert lib.ptcg_embedding_bwd_scratch(1 << 21, 4096, 128) >= 16 << 21


def ln_fwd(lib, x=A, xd=0, ldx=8, gamma=A, beta=A, y=A, yd=0, ldy=8, mean=A, rstd=A, rows=2, width=8):
    return lib.ptcg_layer_norm_fwd(x, xd, ldx, gamma, beta, 1e-5, y, yd, ldy, mean, rstd, rows,
                                   width, None)


@pytest.mark.parametrize("kw", [
    dict(xd=2), dict(yd=7), dict(rows=-1), dict(width=0), dict(width=8193, ldx=9000, ldy=9000),
    dict(ldx=7), dict(ldy=7), dict(x=None), dict(y=None), dict(x=A + 2), dict(gamma=A + 1),
    dict(mean=A + 2)])
def test_layer_norm_refuses(lib, kw):
    assert ln_fwd(lib, **kw) == EINVAL
    assert b"layer norm" in lib.ptcg_last_error()


def test_layer_norm_no_rows(lib):
    assert ln_fwd(lib, rows=0, x=None, y=None) == OK


def ln_bwd(lib, dy=A, dyd=0, lddy=8, x=A, xd=0, ldx=8, mean=A, rstd=A, dres=None, lddres=0, dx=A,
           lddx=8, dgamma=A, dbeta=A, rows=2, width=8, scratch=A, nbytes=1 << 30):
    return lib.ptcg_layer_norm_bwd(dy, dyd, lddy, x, xd, ldx, A, mean, rstd, dres, lddres, dx, lddx,
                                   dgamma, dbeta, 0, rows, width, scratch, nbytes, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(dyd=2), EINVAL), (dict(width=9000), EINVAL), (dict(lddx=4), EINVAL), (dict(dy=None), EINVAL),
    (dict(mean=None), EINVAL), (dict(dx=None), EINVAL), (dict(dgamma=None), EINVAL),
    (dict(dres=A, lddres=4), EINVAL), (dict(dx=A + 2), EINVAL), (dict(scratch=None), ERANGE),
    (dict(nbytes=32), ERANGE)])
def test_layer_norm_gradient_refuses(lib, kw, rc):
    assert ln_bwd(lib, **kw) == rc
    assert b"layer norm gradient" in lib.ptcg_last_error()


def desc(**kw):
    import ptcg_b200.native as n
    d = dict(dtype=1, nseq=2, lq=3, lk=5, heads=4, kv_heads=2, dh=32, scale=0.5)
    strides = {k: kw.pop(k) for k in list(kw) if isinstance(kw[k], tuple)}
    d.update(kw)
    c = n.PtcgCross(**d)
    for name, (l, h) in dict(q=(d["lq"], d["heads"]), out=(d["lq"], d["heads"]),
                             dout=(d["lq"], d["heads"]), dq=(d["lq"], d["heads"]),
                             k=(d["lk"], d["kv_heads"]), v=(d["lk"], d["kv_heads"]),
                             dk=(d["lk"], d["kv_heads"]), dv=(d["lk"], d["kv_heads"])).items():
        s = strides.get(name, (l * h * d["dh"], h * d["dh"], d["dh"]))
        setattr(c, name, n.PtcgHeads(*s))
    return c


def cross_fwd(lib, c, q=A, k=A, v=A, out=A, lse=A, kv_len=None, scratch=A, nbytes=1 << 30):
    return lib.ptcg_cross_attention_fwd(c, q, k, v, None, kv_len, out, lse, scratch, nbytes, None)


def cross_bwd(lib, c, q=A, k=A, v=A, out=A, lse=A, dout=A, dq=A, dk=A, dv=A, scratch=A,
              nbytes=1 << 30):
    return lib.ptcg_cross_attention_bwd(c, q, k, v, None, None, out, lse, dout, dq, dk, dv, scratch,
                                        nbytes, None)


BAD_DESC = [dict(dtype=2), dict(nseq=-1), dict(lq=-1), dict(lk=-1), dict(heads=0), dict(heads=3),
            dict(kv_heads=0), dict(dh=48), dict(dh=256), dict(scale=0.0), dict(scale=-1.0),
            dict(scale=float("inf")), dict(scale=float("nan")), dict(lq=(1 << 30) // 2 + 1)]


@pytest.mark.parametrize("kw", BAD_DESC)
def test_cross_attention_refuses_description(lib, kw):
    c = desc(**kw)
    assert cross_fwd(lib, c) == EINVAL and b"cross attention" in lib.ptcg_last_error()
    assert cross_bwd(lib, c) == EINVAL
    assert lib.ptcg_cross_attention_fwd_scratch(c) == -1
    assert lib.ptcg_cross_attention_bwd_scratch(c) == -1


@pytest.mark.parametrize("kw,args", [
    ({}, dict(q=None)), ({}, dict(k=None)), ({}, dict(v=None)), ({}, dict(out=None)),
    ({}, dict(q=A + 8)), ({}, dict(k=A + 2)), ({}, dict(lse=A + 2)), ({}, dict(kv_len=A + 1)),
    (dict(q=(384, 128, 36)), {}), (dict(k=(320, 68, 32)), {}), (dict(v=(321, 64, 32)), {}),
    (dict(out=(0, 128, 32)), {}), (dict(out=(384, 0, 32)), {}), (dict(out=(384, 128, 16)), {})])
def test_cross_attention_refuses_tensors(lib, kw, args):
    assert cross_fwd(lib, desc(**kw), **args) == EINVAL
    assert b"cross attention" in lib.ptcg_last_error()


@pytest.mark.parametrize("kw,args", [
    ({}, dict(dout=None)), ({}, dict(lse=None)), ({}, dict(dq=None)), ({}, dict(dk=None)),
    ({}, dict(dv=None)), ({}, dict(dk=A + 4)), (dict(dk=(0, 64, 32)), {}), (dict(dv=(320, 64, 0)), {}),
    (dict(dq=(384, 16, 32)), {}), (dict(dout=(384, 129, 32)), {})])
def test_cross_attention_gradient_refuses_tensors(lib, kw, args):
    assert cross_bwd(lib, desc(**kw), **args) == EINVAL
    assert b"cross attention gradient" in lib.ptcg_last_error()


def test_cross_attention_scratch(lib):
    # few rows over a long cache are split, and that needs room for the parts
    c = desc(lq=1, lk=65536)
    need = lib.ptcg_cross_attention_fwd_scratch(c)
    assert need > 0
    assert cross_fwd(lib, c, nbytes=need - 1) == ERANGE
    assert cross_fwd(lib, c, scratch=None) == ERANGE
    assert lib.ptcg_cross_attention_fwd_scratch(desc(nseq=1000)) == 0
    # the gradient always keeps delta there
    assert cross_bwd(lib, desc(), scratch=None) == ERANGE
    assert cross_bwd(lib, desc(), nbytes=8) == ERANGE


def test_cross_attention_nothing_to_do(lib):
    assert cross_fwd(lib, desc(nseq=0), q=None, out=None) == OK
    assert cross_fwd(lib, desc(lq=0), q=None, out=None) == OK
    assert cross_bwd(lib, desc(nseq=0), q=None, dq=None) == OK


# ---------------------------------------------------------- torch-facing
def test_torch_calls_refuse(pkg):
    import ptcg_b200.ops as ops
    from ptcg_b200.native import PtcgError
    t, i32 = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int32)
    q, k = torch.zeros(2, 3, 4, 32), torch.zeros(2, 5, 2, 32)
    o, lse = torch.zeros(2, 3, 4, 32), torch.zeros(2, 4, 3)
    one = torch.zeros(8)
    for call in [
            lambda: ops.embedding(t, i32),                                   # not on a GPU
            lambda: ops.embedding(t, i32.long()),
            lambda: ops.embedding(t[0], i32),
            lambda: ops.embedding(t, i32, pad_id=-3),
            lambda: ops.embedding(t.half(), i32),
            lambda: ops.embedding(t, i32, out_dtype=torch.float16),
            lambda: ops.embedding_backward(torch.zeros(2, 8), i32, 4),
            lambda: ops.embedding_backward(torch.zeros(3, 8), i32, 4, accumulate=True),
            lambda: ops.embedding_backward(torch.zeros(3, 8), i32, 4, dtable=torch.zeros(4, 9)),
            lambda: ops.embedding_backward(torch.zeros(3, 8), i32, 0),
            lambda: ops.layer_norm(t, one, one),
            lambda: ops.layer_norm(torch.tensor(1.0)),
            lambda: ops.layer_norm(t, torch.zeros(7)),
            lambda: ops.layer_norm(t, one.bfloat16()),
            lambda: ops.layer_norm_backward(t, t[:3], one, one[:4], one[:4]),
            lambda: ops.layer_norm_backward(t, t, one, one[:4], one[:4], dres=t.bfloat16()),
            lambda: ops.layer_norm_backward(t, t, one, one[:3], one[:4]),
            lambda: ops.layer_norm_backward(t, t, one, one[:4], one[:4], accumulate=True),
            lambda: ops.layer_norm_backward(t, t, one, one[:4], one[:4], dgamma=one),
            lambda: ops.cross_attention(q, k, k),
            lambda: ops.cross_attention(q, k, k[:, :4]),
            lambda: ops.cross_attention(q, k.bfloat16(), k),
            lambda: ops.cross_attention(q[0], k, k),
            lambda: ops.cross_attention(q, k, k, keep=torch.ones(2, 4, dtype=torch.bool)),
            lambda: ops.cross_attention(q, k, k, keep=torch.ones(2, 5)),
            lambda: ops.cross_attention(q, k, k, kv_len=torch.ones(2, dtype=torch.int64)),
            lambda: ops.cross_attention(q, k, k, scale=-1.0),
            lambda: ops.cross_attention(q.expand(2, 3, 4, 32)[..., :16], k[..., :16], k[..., :16]),
            lambda: ops.cross_attention_backward(o[:1], q, k, k, o, lse),
            lambda: ops.cross_attention_backward(o, q, k, k, o, lse.double()),
            lambda: ops.cross_attention_backward(o, q, k, k, o.bfloat16(), lse)]:
        with pytest.raises(PtcgError):
            call()


def test_torch_calls_refuse_missing_statistics(pkg):
    """What layer_norm(stats=False) returns is no argument of the backward."""
    import ptcg_b200.ops as ops
    from ptcg_b200.native import PtcgError
    t, s, one = torch.zeros(4, 8), torch.zeros(4), torch.zeros(8)
    q, k = torch.zeros(2, 3, 4, 32), torch.zeros(2, 5, 2, 32)
    for call in [lambda: ops.layer_norm_backward(t, t, one, None, None),
                 lambda: ops.layer_norm_backward(t, t, one, s, None),
                 lambda: ops.layer_norm_backward(t, t, one, None, s, weight_grads=False),
                 lambda: ops.cross_attention_backward(q, q, k, k, q, None)]:
        with pytest.raises(PtcgError, match="not None"):
            call()


def test_torch_calls_refuse_sizes_past_32_bits(pkg):
    """They are ints in C, and what is above 2^31 would be cut off."""
    import ptcg_b200.ops as ops
    from ptcg_b200.native import PtcgError
    big = (1 << 32) + 5
    i32, one = torch.zeros(3, dtype=torch.int32), torch.zeros(1)
    q, k = torch.zeros(1, 1, 1, 32), torch.zeros(1, 1, 1, 32)
    row = one.expand(big)
    for call in [lambda: ops.embedding(torch.zeros(4, 8), i32, pad_id=big),
                 lambda: ops.embedding(torch.zeros(4, 8), i32, pad_id=1 << 31),
                 lambda: ops.embedding(one.expand(big, 1), i32),
                 lambda: ops.embedding(one.expand(1, big), i32),
                 lambda: ops.embedding_backward(torch.zeros(3, 8), i32, big),
                 lambda: ops.embedding_backward(torch.zeros(3, 8), i32, 4, pad_id=big),
                 lambda: ops.embedding_backward(one.expand(3, big), i32, 4),
                 lambda: ops.layer_norm(row),
                 lambda: ops.layer_norm_backward(row, row, None, one, one),
                 lambda: ops.cross_attention(q, k.expand(1, big, 1, 32), k.expand(1, big, 1, 32)),
                 lambda: ops.cross_attention(q.expand(1, big, 1, 32), k, k),
                 lambda: ops.cross_attention(q.expand(big, 1, 1, 32), *[k.expand(big, 1, 1, 32)] * 2)]:
        with pytest.raises(PtcgError, match="32 bits"):
            call()
    with pytest.raises(PtcgError, match="at least 1"):
        ops.embedding_backward(torch.zeros(3, 8), i32, -1)


def test_torch_calls_refuse_what_autograd_would_lose(pkg):
    import ptcg_b200.ops as ops
    from ptcg_b200.native import PtcgError
    z = lambda *s, need=False: torch.zeros(*s, requires_grad=need)     # noqa: E731
    i32, s, one, lse = torch.zeros(3, dtype=torch.int32), z(4), z(8), z(2, 4, 3)
    q, k, t = z(2, 3, 4, 32), z(2, 5, 2, 32), z(4, 8)
    calls = [lambda n: ops.embedding(z(4, 8, need=n), i32),
             lambda n: ops.embedding_backward(z(3, 8, need=n), i32, 4),
             lambda n: ops.layer_norm(z(4, 8, need=n)),
             lambda n: ops.layer_norm(t, z(8, need=n)),
             lambda n: ops.layer_norm(t, one, z(8, need=n)),
             lambda n: ops.layer_norm_backward(z(4, 8, need=n), t, one, s, s),
             lambda n: ops.layer_norm_backward(t, t, one, s, s, dres=z(4, 8, need=n)),
             lambda n: ops.cross_attention(z(2, 3, 4, 32, need=n), k, k),
             lambda n: ops.cross_attention(q, z(2, 5, 2, 32, need=n), k),
             lambda n: ops.cross_attention(q, k, z(2, 5, 2, 32, need=n)),
             lambda n: ops.cross_attention_backward(z(2, 3, 4, 32, need=n), q, k, k, q, lse)]
    for call in calls:
        with pytest.raises(PtcgError, match="records? nothing for autograd"):
            call(True)
        with pytest.raises(PtcgError, match="CUDA"):                   # past that check
            call(False)
        with torch.no_grad(), pytest.raises(PtcgError, match="CUDA"):
            call(True)


def test_cross_attention_refuses_scales_that_overflow_in_base_2(lib):
    c = desc(scale=3e38)
    assert cross_fwd(lib, c) == EINVAL and b"scale" in lib.ptcg_last_error()
    assert cross_bwd(lib, c) == EINVAL and lib.ptcg_cross_attention_fwd_scratch(c) == -1
    assert lib.ptcg_cross_attention_fwd_scratch(desc(scale=2e38)) >= 0
