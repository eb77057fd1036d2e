"""Torch-facing calls of the decoder operators (include/ptcg_b200.h): embedding
lookup, layer norm and cross attention to an encoder's states, each with its
backward pass.

Tensors are torch CUDA tensors of one device, fp32 or bf16; the work is
enqueued on that device's current stream, on outputs and scratch that come
from torch's allocator.  Nothing waits on the host, so the calls can be
captured in a CUDA graph.  A tensor last used on another stream has to be
ordered before the call by the caller, as for any torch operation.  Arguments
are checked before anything is launched; errors raise `PtcgError`.  Nothing is
recorded for autograd: the gradients are calls of their own.  A forward whose
inputs, or a backward whose incoming gradients, require grad is refused while
autograd records (its outputs would be cut off without a word); under
`torch.no_grad()`, in an `autograd.Function` and on detached tensors they run.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import native
from .native import PtcgCross, PtcgError, PtcgHeads, check

_DT = {torch.float32: 0, torch.bfloat16: 1}
_BYTES = (torch.bool, torch.uint8)


def _bad(msg):
    raise PtcgError(msg)


def _records_nothing(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                _bad("an input requires grad, but the operators record nothing for autograd: "
                     "call them under torch.no_grad() or on detached tensors")


def _fits(what, *sizes):
    """The C entries take these as 32-bit ints; ctypes would cut them off."""
    if max(sizes) > 0x7fffffff:
        _bad(f"{what}: sizes {sizes} do not all fit 32 bits")


def _dt(t, what):
    d = _DT.get(t.dtype)
    if d is None:
        _bad(f"{what}: dtype {t.dtype} is neither float32 nor bfloat16")
    return d


def _on(dev, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            _bad(f"{name} is on {t.device}, not on {dev}")


def _f32(dev, shape, **tensors):
    for name, t in tensors.items():
        if t is None:
            continue
        if t.dtype != torch.float32 or t.device != dev or t.shape != shape or not t.is_contiguous():
            _bad(f"{name} must be a contiguous float32 tensor of shape {shape} on {dev}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(dev, fn, *args):
    """fn(*args, stream) with `dev` current, on its current stream (the raw
    handle: a Stream object costs as much as the launch)."""
    if dev.type != "cuda":
        _bad("the operators run on CUDA tensors")
    i = dev.index
    if torch.cuda.current_device() == i:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    if rc:
        check(rc)


def _rows(t, width, what):
    """(tensor as rows of `width` contiguous elements, rows, pitch); a copy only
    where the leading dimensions have no common pitch."""
    shape = t.shape
    if not shape or shape[-1] != width:
        _bad(f"{what}: last dimension must be {width}, got shape {tuple(shape)}")
    if t.is_contiguous():
        return t, t.numel() // width if width else 0, width
    if len(shape) != 2:
        t = t.reshape(-1, width)
    if width > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < width:
        t = t.contiguous()
    n = t.shape[0]
    return t, n, (t.stride(0) if n > 1 else width)


def _scratch(nbytes, dev):
    if nbytes < 0:
        _bad(native.lib().ptcg_last_error().decode())
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


# -------------------------------------------------------------- embedding
def _ids(ids, dev):
    if ids.dtype != torch.int32 or ids.device != dev:
        _bad(f"ids must be an int32 tensor on {dev}, got {ids.dtype} on {ids.device}")
    return ids.contiguous()


def _pad(pad_id):
    if pad_id is None:
        return -1
    if not 0 <= pad_id <= 0x7fffffff:
        _bad(f"pad_id {pad_id} must be None or an id of 32 bits, at least 0")
    return int(pad_id)


def embedding(table, ids, scale=1.0, pad_id=None, out_dtype=None):
    """scale * table[ids] -> ids.shape + (width,) in out_dtype (the table's by
    default).  Ids are clamped to the table; places whose id is pad_id give
    zeros."""
    if table.dim() != 2:
        _bad("table must be (vocab, width)")
    _records_nothing(table)
    dev = table.device
    vocab, width = table.shape
    _fits("table", vocab, width)
    pad_id = _pad(pad_id)
    ids = _ids(ids, dev)
    tab, _, ldt = _rows(table, width, "table")
    out = torch.empty(*ids.shape, width, dtype=out_dtype or table.dtype, device=dev)
    _call(dev, native.lib().ptcg_embedding_fwd, tab.data_ptr(), _dt(table, "table"), ldt, vocab,
          width, ids.data_ptr(), ids.numel(), scale, pad_id, out.data_ptr(),
          _dt(out, "out"), width)
    return out


def embedding_backward(dout, ids, vocab, scale=1.0, pad_id=None, dtable=None, accumulate=False):
    """Gradient of `embedding` for its table: float32 (vocab, width), every row
    the sum of its places' gradients, in an order that follows from the ids
    alone.  With accumulate, added to dtable."""
    _records_nothing(dout)
    dev = dout.device
    ids = _ids(ids, dev)
    if dout.dim() != ids.dim() + 1 or dout.shape[:-1] != ids.shape:
        _bad(f"dout {tuple(dout.shape)} does not match ids {tuple(ids.shape)}")
    width = dout.shape[-1]
    _fits("dout", vocab, width)
    if vocab <= 0:
        _bad(f"vocab {vocab} must be at least 1")
    pad_id = _pad(pad_id)
    g, n, ldg = _rows(dout, width, "dout")
    if dtable is None:
        if accumulate:
            _bad("accumulate needs dtable")
        dtable = torch.empty(vocab, width, device=dev)
    elif (dtable.dtype != torch.float32 or dtable.device != dev or dtable.shape != (vocab, width)
          or (width > 1 and dtable.stride(1) != 1) or (vocab > 1 and dtable.stride(0) < width)):
        _bad(f"dtable must be float32 rows of shape {(vocab, width)} on {dev}")
    lib = native.lib()
    nbytes = lib.ptcg_embedding_bwd_scratch(n, vocab, width)
    scratch = _scratch(nbytes, dev)
    _call(dev, lib.ptcg_embedding_bwd, g.data_ptr(), _dt(dout, "dout"), ldg, ids.data_ptr(), n,
          scale, pad_id, dtable.data_ptr(), dtable.stride(0) if vocab > 1 else width, vocab,
          width, int(accumulate), _ptr(scratch), nbytes)
    return dtable


# ------------------------------------------------------------- layer norm
def layer_norm(x, gamma=None, beta=None, eps=1e-5, out_dtype=None, stats=True):
    """(y, mean, rstd) of a layer norm over the last dimension; gamma / beta
    float32 or None (1 / 0).  mean and rstd (float32, x.shape[:-1]) are what
    the backward takes; stats=False leaves them out (None)."""
    _records_nothing(x, gamma, beta)
    dev, width = x.device, x.shape[-1] if x.dim() else 0
    _fits("x", width)
    xr, n, ldx = _rows(x, width, "x")
    _f32(dev, (width,), gamma=gamma, beta=beta)
    y = torch.empty(*x.shape, dtype=out_dtype or x.dtype, device=dev)
    mean = torch.empty(x.shape[:-1], device=dev) if stats else None
    rstd = torch.empty(x.shape[:-1], device=dev) if stats else None
    _call(dev, native.lib().ptcg_layer_norm_fwd, xr.data_ptr(), _dt(x, "x"), ldx, _ptr(gamma),
          _ptr(beta), eps, y.data_ptr(), _dt(y, "y"), width, _ptr(mean), _ptr(rstd), n, width)
    return y, mean, rstd


def layer_norm_backward(dy, x, gamma, mean, rstd, dres=None, dgamma=None, dbeta=None,
                        accumulate=False, weight_grads=True):
    """(dx, dgamma, dbeta) of `layer_norm`; dx in x's type, plus dres (the
    gradient that reaches x past the norm, x's type) if given.  dgamma / dbeta
    are new, or written or (accumulate) added to where given; with
    weight_grads=False they are None."""
    _records_nothing(dy, dres)
    dev, width = x.device, x.shape[-1] if x.dim() else 0
    _fits("x", width)
    if mean is None or rstd is None:
        _bad("mean and rstd are the forward's (layer_norm with stats=True), not None")
    xr, n, ldx = _rows(x, width, "x")
    if dy.shape != x.shape or (dres is not None and (dres.shape != x.shape or dres.dtype != x.dtype)):
        _bad("dy and dres must have x's shape, and dres its type")
    _on(dev, dy=dy, dres=dres)
    gr, _, ldg = _rows(dy, width, "dy")
    rr, _, ldr = _rows(dres, width, "dres") if dres is not None else (None, 0, 0)
    _f32(dev, (width,), gamma=gamma, dgamma=dgamma, dbeta=dbeta)
    _f32(dev, x.shape[:-1], mean=mean, rstd=rstd)
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
    if not weight_grads:
        if dgamma is not None or dbeta is not None:
            _bad("weight_grads=False takes no dgamma / dbeta")
    elif dgamma is None or dbeta is None:
        if accumulate or dgamma is not None or dbeta is not None:
            _bad("give both dgamma and dbeta (accumulate needs them), or neither")
        dgamma, dbeta = torch.empty(2, width, device=dev)
    lib = native.lib()
    nbytes = lib.ptcg_layer_norm_bwd_scratch(n, width) if weight_grads else 0
    scratch = _scratch(nbytes, dev)
    _call(dev, lib.ptcg_layer_norm_bwd, gr.data_ptr(), _dt(dy, "dy"), ldg, xr.data_ptr(),
          _dt(x, "x"), ldx, _ptr(gamma), mean.data_ptr(), rstd.data_ptr(), _ptr(rr), ldr,
          dx.data_ptr(), width, _ptr(dgamma), _ptr(dbeta), int(accumulate), n, width,
          _ptr(scratch), nbytes)
    return dx, dgamma, dbeta


# -------------------------------------------------------- cross attention
@functools.lru_cache(maxsize=256)
def _cross(dtype, dims, scale, strides, backward):
    """The C description of a problem (plain sizes and strides, no addresses)
    and the bytes of scratch it needs."""
    c = PtcgCross(dtype, *dims, scale, *[PtcgHeads(*s) for s in strides])
    lib = native.lib()
    nbytes = (lib.ptcg_cross_attention_bwd_scratch if backward
              else lib.ptcg_cross_attention_fwd_scratch)(c)
    if nbytes < 0:
        _bad(lib.ptcg_last_error().decode())
    return c, nbytes


_ZERO = (0, 0, 0)


def _head_strides(t, what):
    a, b, c, d = t.stride()
    n, r, h, w = t.shape
    if d != 1 and w > 1:
        _bad(f"{what}: the head's elements must be contiguous, got strides {t.stride()}")
    # a dimension of one element has no stride that matters
    return a if n > 1 else 0, b if r > 1 else 0, c if h > 1 else 0


def _cross_args(q, k, v, keep, kv_len, scale):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        _bad("q, k and v must be (nseq, rows, heads, width)")
    dev, dt = q.device, _dt(q, "q")
    nseq, lq, heads, dh = q.shape
    lk, kvh = k.shape[1], k.shape[2]
    _fits("q, k", nseq, lq, lk, heads, kvh, dh)
    if k.shape[0] != nseq or k.shape[3] != dh or v.shape != k.shape:
        _bad(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        _bad("q, k and v must have one type")
    if k.device != dev or v.device != dev:
        _on(dev, k=k, v=v)
    if keep is not None:
        if keep.shape != (nseq, lk) or keep.dtype not in _BYTES or keep.device != dev:
            _bad(f"keep must be a bool or uint8 tensor of shape {(nseq, lk)} on {dev}")
        keep = keep.contiguous()
    if kv_len is not None:
        if kv_len.shape != (nseq,) or kv_len.dtype != torch.int32 or kv_len.device != dev:
            _bad(f"kv_len must be an int32 tensor of shape {(nseq,)} on {dev}")
        kv_len = kv_len.contiguous()
    scale = dh ** -0.5 if scale is None else float(scale)
    return dev, dt, (nseq, lq, lk, heads, kvh, dh), keep, kv_len, scale


def cross_attention(q, k, v, keep=None, kv_len=None, scale=None):
    """(out, lse): q (nseq, lq, heads, dh) attends to k, v (nseq, lk, kv_heads,
    dh), any strides with a contiguous head and 16-byte aligned rows.  keep
    (nseq, lk) bool / uint8 and kv_len (nseq,) int32 mask keys; scale defaults
    to dh ** -0.5.  out is q's shape and type; lse (nseq, heads, lq) float32
    is what the backward takes (-inf, with out 0, where no key is kept)."""
    _records_nothing(q, k, v)
    dev, dt, dims, keep, kv_len, scale = _cross_args(q, k, v, keep, kv_len, scale)
    nseq, lq, lk, heads, kvh, dh = dims
    out = torch.empty(nseq, lq, heads, dh, dtype=q.dtype, device=dev)
    lse = torch.empty(nseq, heads, lq, device=dev)
    c, nbytes = _cross(dt, dims, scale, (_head_strides(q, "q"), _head_strides(k, "k"),
                                         _head_strides(v, "v"), (lq * heads * dh, heads * dh, dh),
                                         _ZERO, _ZERO, _ZERO, _ZERO), False)
    scratch = _scratch(nbytes, dev)
    _call(dev, native.lib().ptcg_cross_attention_fwd, c, q.data_ptr(), k.data_ptr(), v.data_ptr(),
          _ptr(keep), _ptr(kv_len), out.data_ptr(), lse.data_ptr(), _ptr(scratch), nbytes)
    return out, lse


def cross_attention_backward(dout, q, k, v, out, lse, keep=None, kv_len=None, scale=None):
    """(dq, dk, dv) of `cross_attention`, contiguous, in the inputs' type and
    shapes; out and lse are the forward's.  dk and dv are summed over the query
    heads of a group and are zero for masked keys."""
    _records_nothing(dout)
    dev, dt, dims, keep, kv_len, scale = _cross_args(q, k, v, keep, kv_len, scale)
    nseq, lq, lk, heads, kvh, dh = dims
    if dout.shape != q.shape or out.shape != q.shape or dout.dtype != q.dtype or out.dtype != q.dtype:
        _bad("dout and out must have q's shape and type")
    _on(dev, dout=dout, out=out)
    if lse is None:
        _bad("lse is the forward's, not None")
    _f32(dev, (nseq, heads, lq), lse=lse)
    dq = torch.empty(nseq, lq, heads, dh, dtype=q.dtype, device=dev)
    dk = torch.empty(nseq, lk, kvh, dh, dtype=q.dtype, device=dev)
    dv = torch.empty(nseq, lk, kvh, dh, dtype=q.dtype, device=dev)
    sq, sk = (lq * heads * dh, heads * dh, dh), (lk * kvh * dh, kvh * dh, dh)
    c, nbytes = _cross(dt, dims, scale, (_head_strides(q, "q"), _head_strides(k, "k"),
                                         _head_strides(v, "v"), _head_strides(out, "out"),
                                         _head_strides(dout, "dout"), sq, sk, sk), True)
    scratch = _scratch(nbytes, dev)
    _call(dev, native.lib().ptcg_cross_attention_bwd, c, q.data_ptr(), k.data_ptr(), v.data_ptr(),
          _ptr(keep), _ptr(kv_len), out.data_ptr(), lse.data_ptr(), dout.data_ptr(),
          dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(scratch), nbytes)
    return dq, dk, dv
