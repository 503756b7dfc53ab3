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


def _tensor(x, name, like=None, shape=None):
    if not isinstance(x, torch.Tensor) or x.dim() != 4:
        _bad("%s must be a [batch, row, head, dim] tensor" % name)
    if like is not None and (x.dtype != like.dtype or x.device != like.device):
        _bad("%s must have the type and device of q" % name)
    if shape is not None and tuple(x.shape) != shape:
        _bad("%s must be of shape %s, not %s" % (name, list(shape), list(x.shape)), E_SIZE_MISMATCH)
    return x


def _usable(x, group=1):
    """x itself, or a copy when the kernels cannot address it (gpx_view in include/gpx.h)."""
    if x.numel() == 0:
        return x
    m = 16 // x.element_size()
    b, r, h, d = x.stride()
    if d != 1 or b % m or r % m or h % m or x.data_ptr() % 16 or (r < x.shape[3] and x.shape[1] > 1) or r > 1 << 22 or h * group > 1 << 27:
        # clone: .contiguous() would hand back an offset view that is contiguous but not aligned
        return x.clone(memory_format=torch.contiguous_format)
    return x


def _view(x):
    b, r, h, _ = x.stride()
    return (x.data_ptr(), b, r, h)


def _lengths(x, name, n, device):
    if x is None:
        return 0
    if not isinstance(x, torch.Tensor) or x.dtype != torch.int32 or x.dim() != 1 or x.device != device or not x.is_contiguous():
        _bad("%s must be a contiguous int32 tensor [batch] on the device of q" % name)
    if x.shape[0] != n:
        _bad("%s must have one entry per batch member" % name, E_SIZE_MISMATCH)
    return x.data_ptr()


def _mask(x, batch, nk, device):
    if x is None:
        return 0, 0
    if not isinstance(x, torch.Tensor) or x.dtype not in (torch.bool, torch.uint8) or x.device != device or x.dim() != 2 or \
            (x.numel() and x.stride(1) != 1 and nk != 1):
        _bad("key_mask must be a bool tensor [batch, nk] on the device of q, its rows contiguous")
    if tuple(x.shape) != (batch, nk):
        _bad("key_mask must be of shape %s, not %s" % ([batch, nk], list(x.shape)), E_SIZE_MISMATCH)
    return x.data_ptr(), x.stride(0)


def _queries(q, k, scale):
    _tensor(q, "q")
    if q.dtype not in _SCALARS:
        _bad("q must be float32, float16 or bfloat16")
    if not q.is_cuda:
        _bad("q must be on a GPU: libgpx has no CPU path")
    b, nq, hq, d = q.shape
    hk = k.shape[-2]
    if hk < 1 or hq < 1 or hq % hk:
        _bad("the key heads must divide the query heads")
    if d < 8 or d > MAX_DIM or d % 8:
        _bad("dim must be a multiple of 8 up to %d" % MAX_DIM)
    scale = d ** -0.5 if scale is None else float(scale)
    return b, nq, hq, hk, d, scale


def _run(which, q, sizes, scale, views, lse, lens, mask, grads, own, own_len):
    device = q.device
    stream = torch.cuda.current_stream(device).cuda_stream
    head = (_SCALARS[q.dtype], device.index) + sizes + (scale,) + views + (lse,) + lens + mask + grads + own + (own_len,)
    need = C.c_size_t(0)
    args = _ARGS.pack(*head, 0, 0, stream)
    _check(_entry(3)(args, which, C.byref(need)))
    if need.value:
        work = torch.empty(need.value, dtype=torch.uint8, device=device)
        args = _ARGS.pack(*head, work.data_ptr(), need.value, stream)
    _check(_entry(which)(args))


def attend(q, k, v, scale=None, k_len=None, key_mask=None, q_len=None):
    """o [batch, nq, heads, dim] and lse [batch, heads, nq] (float32) of queries q [batch, nq, heads, dim] over k, v
    [batch, nk, heads_kv, dim].  scale: dim ** -0.5 unless given.  k_len, q_len: int32 [batch], entries and queries that count
    (the others' o is zero, lse -inf); key_mask: bool [batch, nk], True where the entry counts."""
    _tensor(k, "k")
    b, nq, hq, hk, d, scale = _queries(q, k, scale)
    nk = k.shape[1]
    _tensor(k, "k", q, (b, nk, hk, d))
    _tensor(v, "v", q, (b, nk, hk, d))
    lens = (_lengths(q_len, "q_len", b, q.device), _lengths(k_len, "k_len", b, q.device))
    mask = _mask(key_mask, b, nk, q.device)
    q, k, v = _usable(q, hq // hk), _usable(k), _usable(v)
    o = torch.empty((b, nq, hq, d), dtype=q.dtype, device=q.device)
    lse = torch.empty((b, hq, nq), dtype=torch.float32, device=q.device)
    _run(FORWARD, q, (b, nq, nk, 0, hq, hk, d), scale, _view(q) + _view(k) + _view(v) + _view(o), lse.data_ptr(), lens, mask,
         _NONE * 4, _NONE * 2, 0)
    return o, lse


def attend_backward(d_o, q, k, v, o, lse, scale=None, k_len=None, key_mask=None, q_len=None):
    """dq, dk, dv for the gradient d_o of attend's o; o and lse as attend returned them, the other arguments as it got them."""
    _tensor(k, "k")
    b, nq, hq, hk, d, scale = _queries(q, k, scale)
    nk = k.shape[1]
    _tensor(k, "k", q, (b, nk, hk, d))
    _tensor(v, "v", q, (b, nk, hk, d))
    _tensor(o, "o", q, (b, nq, hq, d))
    _tensor(d_o, "d_o", q, (b, nq, hq, d))
    if not isinstance(lse, torch.Tensor) or lse.dtype != torch.float32 or lse.device != q.device or not lse.is_contiguous():
        _bad("lse must be a contiguous float32 tensor on the device of q")
    if tuple(lse.shape) != (b, hq, nq):
        _bad("lse must be of shape %s, not %s" % ([b, hq, nq], list(lse.shape)), E_SIZE_MISMATCH)
    lens = (_lengths(q_len, "q_len", b, q.device), _lengths(k_len, "k_len", b, q.device))
    mask = _mask(key_mask, b, nk, q.device)
    q, k, v, o, d_o = _usable(q, hq // hk), _usable(k), _usable(v), _usable(o), _usable(d_o, hq // hk)
    dq = torch.empty((b, nq, hq, d), dtype=q.dtype, device=q.device)
    dk = torch.empty((b, nk, hk, d), dtype=q.dtype, device=q.device)
    dv = torch.empty((b, nk, hk, d), dtype=q.dtype, device=q.device)
    _run(BACKWARD, q, (b, nq, nk, 0, hq, hk, d), scale, _view(q) + _view(k) + _view(v) + _view(o), lse.data_ptr(), lens, mask,
         _view(d_o) + _view(dq) + _view(dk) + _view(dv), _NONE * 2, 0)
    return dq, dk, dv


def attend_shared(q, k, v, k_own, v_own, own_len=None, scale=None):
    """o and lse (as attend) of a batch over ONE context: q [batch, nq, heads, dim]; k, v [nk, heads_kv, dim], which every query
    sees; k_own, v_own [batch, n_own, heads_kv, dim], of which own_len[b] (int32 [batch]; None: all) exist, the rows of the nq
    queries last: query i sees the own entries j < own_len[b] - (nq - 1 - i).  The context is read once for the whole batch."""
    if not isinstance(k, torch.Tensor) or k.dim() != 3 or not isinstance(v, torch.Tensor) or v.dim() != 3:
        _bad("k and v must be [nk, heads_kv, dim] tensors")
    b, nq, hq, hk, d, scale = _queries(q, k, scale)
    nk = k.shape[0]
    k, v = k[None], v[None]
    _tensor(k, "k", q, (1, nk, hk, d))
    _tensor(v, "v", q, (1, nk, hk, d))
    _tensor(k_own, "k_own", q)
    no = k_own.shape[1]
    _tensor(k_own, "k_own", q, (b, no, hk, d))
    _tensor(v_own, "v_own", q, (b, no, hk, d))
    own = _lengths(own_len, "own_len", b, q.device)
    q, k, v, k_own, v_own = _usable(q, hq // hk), _usable(k), _usable(v), _usable(k_own), _usable(v_own)
    o = torch.empty((b, nq, hq, d), dtype=q.dtype, device=q.device)
    lse = torch.empty((b, hq, nq), dtype=torch.float32, device=q.device)
    _run(SHARED, q, (b, nq, nk, no, hq, hk, d), scale, _view(q) + _view(k) + _view(v) + _view(o), lse.data_ptr(), (0, 0), (0, 0),
         _NONE * 4, _view(k_own) + _view(v_own), own)
    return o, lse
