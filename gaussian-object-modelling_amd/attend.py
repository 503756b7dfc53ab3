"""Softmax-weighted sums over a context: gpx_attend, gpx_attend_backward and gpx_attend_shared of include/gpx.h on torch tensors.

The learned-feature counterpart of the predictive mean: queries and context entries carry feature vectors, per head
o_i = sum_j softmax_j(scale <q_i, k_j>) v_j.  Plumbing over the C ABI like gpx.py: torch provides memory, device and stream, every
number comes from the HIP kernels, and there is no CPU fallback.

Tensors are [batch, row, head, dim] of one type (float32, float16 or bfloat16) on one GPU; dim is a multiple of 8 up to 128 and the
key heads divide the query heads.  Strided views are used as they are where gpx_view in include/gpx.h allows it (contiguous dim, base and
strides multiples of 16 bytes); other layouts are copied first.  Work is enqueued on the current stream of the tensors' device.  Gradients are explicit
calls, as for gpx_dgp_loglik_gradient: nothing here is recorded by autograd.
"""
import ctypes as C
import struct

import torch

from .gpx import E_BAD_ARG, E_SIZE_MISMATCH, GpxError, _check, lib

FORWARD, BACKWARD, SHARED = range(3)
MAX_DIM = 128
_SCALARS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ARGS = struct.Struct("@iiqqqqqqqd" + "Pqqq" * 4 + "PPPPq" + "Pqqq" * 6 + "PPQP")  # gpx_attend_args
_NONE = (0, 0, 0, 0)

_calls = None
_workspace = {}  # bytes gpx_attend_workspace gave for (call, scalar, device, sizes, scale)


def _entry(which):
    global _calls
    if _calls is None:
        L = lib()
        for f in (L.gpx_attend, L.gpx_attend_backward, L.gpx_attend_shared):
            f.restype, f.argtypes = C.c_int, [C.c_char_p]
        L.gpx_attend_workspace.restype, L.gpx_attend_workspace.argtypes = C.c_int, [C.c_char_p, C.c_int, C.POINTER(C.c_size_t)]
        _calls = (L.gpx_attend, L.gpx_attend_backward, L.gpx_attend_shared, L.gpx_attend_workspace)
    return _calls[which]


def _bad(msg, code=E_BAD_ARG):
    raise GpxError(code, msg)


def _queries(q, hk, scale):
    """The checks of q -> (batch, nq, heads, dim, scale)."""
    if not isinstance(q, torch.Tensor) or q.dim() != 4:
        _bad("q must be a [batch, row, head, dim] tensor")
    if q.dtype not in _SCALARS:
        _bad("q must be float32, float16 or bfloat16")
    if not q.is_cuda:
        _bad("q must be on a GPU: libgpx has no CPU path")
    b, nq, hq, d = q.shape
    if hk < 1 or hq < 1 or hq % hk:
        _bad("the key heads must divide the query heads")
    if d < 8 or d > MAX_DIM or d % 8:
        _bad("dim must be a multiple of 8 up to %d" % MAX_DIM)
    return b, nq, hq, d, d ** -0.5 if scale is None else float(scale)


def _heads(k, dims):
    if not isinstance(k, torch.Tensor) or k.dim() != dims:
        _bad("keys must be a %s tensor" % ("[batch, row, head, dim]" if dims == 4 else "[row, head, dim]"))
    return k.shape[dims - 2]


def _operand(x, name, q, shape, group=1):
    """x and its gpx_view; a copy of x where the kernels cannot address it (gpx_view in include/gpx.h)."""
    if not isinstance(x, torch.Tensor) or x.dtype != q.dtype or x.device != q.device:
        _bad("%s must be a tensor of the type and device of q" % name)
    if x.shape != shape:
        _bad("%s must be of shape %s, not %s" % (name, list(shape), list(x.shape)), E_SIZE_MISMATCH)
    b, r, h, d = x.stride()
    p = x.data_ptr()
    if (p | (b | r | h) * x.element_size()) & 15 or d != 1 or r > 1 << 22 or h * group > 1 << 27 or (r < shape[3] and shape[1] > 1):
        if x.numel():
            x = x.clone(memory_format=torch.contiguous_format)
            b, r, h, d = x.stride()
            p = x.data_ptr()
    return x, (p, b, r, h)


def _like(x):
    """A contiguous tensor of x's shape, and its gpx_view."""
    y = torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    r, h, d = x.shape[1:]
    return y, (y.data_ptr(), r * h * d, h * d, d)


def _lengths(x, name, q):
    if x is None:
        return 0
    if not isinstance(x, torch.Tensor) or x.dtype != torch.int32 or x.dim() != 1 or x.device != q.device or not x.is_contiguous():
        _bad("%s must be a contiguous int32 tensor [batch] on the device of q" % name)
    if x.shape[0] != q.shape[0]:
        _bad("%s must have one entry per batch member" % name, E_SIZE_MISMATCH)
    return x.data_ptr()


def _mask(x, q, nk):
    if x is None:
        return 0, 0
    if not isinstance(x, torch.Tensor) or x.dtype not in (torch.bool, torch.uint8) or x.device != q.device or x.dim() != 2 or \
            (x.stride(1) != 1 and x.numel() and nk != 1):
        _bad("key_mask must be a bool tensor [batch, nk] on the device of q, its rows contiguous")
    if tuple(x.shape) != (q.shape[0], nk):
        _bad("key_mask must be of shape %s, not %s" % ([q.shape[0], nk], list(x.shape)), E_SIZE_MISMATCH)
    return x.data_ptr(), x.stride(0)


def _run(which, q, rest):
    index = q.device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    head = (_SCALARS[q.dtype], index) + rest
    sizes = (which,) + head[:10]
    need = _workspace.get(sizes)
    if need is None:
        n = C.c_size_t(0)
        _check(_entry(3)(_ARGS.pack(*head, 0, 0, stream), which, C.byref(n)))
        if len(_workspace) >= 4096:
            _workspace.clear()
        need = _workspace[sizes] = n.value
    work = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    rc = _entry(which)(_ARGS.pack(*head, work.data_ptr() if need else 0, need, stream))
    if rc:
        _check(rc)


def attend(q, k, v, scale=None, k_len=None, key_mask=None, q_len=None):
    """o [batch, nq, heads, dim] and lse [batch, heads, nq] (float32) of queries q [batch, nq, heads, dim] over k, v
    [batch, nk, heads_kv, dim].  scale: dim ** -0.5 unless given.  k_len, q_len: int32 [batch], entries and queries that count
    (the others' o is zero, lse -inf); key_mask: bool [batch, nk], True where the entry counts."""
    hk = _heads(k, 4)
    b, nq, hq, d, scale = _queries(q, hk, scale)
    nk = k.shape[1]
    q, qv = _operand(q, "q", q, q.shape, hq // hk)
    k, kv = _operand(k, "k", q, (b, nk, hk, d))
    v, vv = _operand(v, "v", q, (b, nk, hk, d))
    o, ov = _like(q)
    lse = torch.empty((b, hq, nq), dtype=torch.float32, device=q.device)
    _run(FORWARD, q, (b, nq, nk, 0, hq, hk, d, scale) + qv + kv + vv + ov
         + (lse.data_ptr(), _lengths(q_len, "q_len", q), _lengths(k_len, "k_len", q)) + _mask(key_mask, q, nk) + _NONE * 6 + (0,))
    return o, lse


def attend_backward(d_o, q, k, v, o, lse, scale=None, k_len=None, key_mask=None, q_len=None):
    """dq, dk, dv for the gradient d_o of attend's o; o and lse as attend returned them, the other arguments as it got them."""
    hk = _heads(k, 4)
    b, nq, hq, d, scale = _queries(q, hk, scale)
    nk = k.shape[1]
    q, qv = _operand(q, "q", q, q.shape, hq // hk)
    k, kv = _operand(k, "k", q, (b, nk, hk, d))
    v, vv = _operand(v, "v", q, (b, nk, hk, d))
    o, ov = _operand(o, "o", q, (b, nq, hq, d))
    d_o, gv = _operand(d_o, "d_o", q, (b, nq, hq, d), hq // hk)
    if not isinstance(lse, torch.Tensor) or lse.dtype != torch.float32 or lse.device != q.device or not lse.is_contiguous():
        _bad("lse must be a contiguous float32 tensor on the device of q")
    if lse.shape != (b, hq, nq):
        _bad("lse must be of shape %s, not %s" % ([b, hq, nq], list(lse.shape)), E_SIZE_MISMATCH)
    dq, dqv = _like(q)
    dk, dkv = _like(k)
    dv, dvv = _like(v)
    _run(BACKWARD, q, (b, nq, nk, 0, hq, hk, d, scale) + qv + kv + vv + ov
         + (lse.data_ptr(), _lengths(q_len, "q_len", q), _lengths(k_len, "k_len", q)) + _mask(key_mask, q, nk)
         + gv + dqv + dkv + dvv + _NONE * 2 + (0,))
    return dq, dk, dv


def attend_shared(q, k, v, k_own, v_own, own_len=None, scale=None):
    """o and lse (as attend) of a batch over ONE context: q [batch, nq, heads, dim]; k, v [nk, heads_kv, dim], which every query
    sees; k_own, v_own [batch, n_own, heads_kv, dim], of which own_len[b] (int32 [batch]; None: all) exist, the rows of the nq
    queries last: query i sees the own entries j < own_len[b] - (nq - 1 - i).  The context is read once for the whole batch."""
    hk = _heads(k, 3)
    if _heads(v, 3) != hk or _heads(k_own, 4) != hk:
        _bad("k, v, k_own and v_own must have the same heads", E_SIZE_MISMATCH)
    b, nq, hq, d, scale = _queries(q, hk, scale)
    nk, no = k.shape[0], k_own.shape[1]
    q, qv = _operand(q, "q", q, q.shape, hq // hk)
    k, kv = _operand(k[None], "k", q, (1, nk, hk, d))
    v, vv = _operand(v[None], "v", q, (1, nk, hk, d))
    k_own, kov = _operand(k_own, "k_own", q, (b, no, hk, d))
    v_own, vov = _operand(v_own, "v_own", q, (b, no, hk, d))
    o, ov = _like(q)
    lse = torch.empty((b, hq, nq), dtype=torch.float32, device=q.device)
    _run(SHARED, q, (b, nq, nk, no, hq, hk, d, scale) + qv + kv + vv + ov + (lse.data_ptr(), 0, 0, 0, 0) + _NONE * 4 + kov + vov
         + (_lengths(own_len, "own_len", q),))
    return o, lse
