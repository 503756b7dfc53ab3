"""Softmax-weighted sums over a context: gpx_attend, gpx_attend_backward and gpx_attend_shared of include/gpx.h on torch tensors.

The learned-feature counterpart of the predictive mean: queries and context entries carry feature vectors, per head
o_i = sum_j softmax_j(scale <q_i, k_j>) v_j.  Plumbing over the C ABI like gpx.py: torch provides memory, device and stream, every
number comes from the HIP kernels, and there is no CPU fallback.  Checks and allocations are in csrc/gpx_torch.cpp.

Tensors are [batch, row, head, dim] of one type (float32, float16 or bfloat16) on one GPU; dim is a multiple of 8 up to 128 and the
key heads divide the query heads.  Strided views are used as they are where gpx_view in include/gpx.h allows it (contiguous dim,
base and strides multiples of 16 bytes); other layouts are copied first.  Work is enqueued on the current stream of the tensors'
device.  What a call refuses raises GpxError.  Gradients are explicit calls, as for gpx_dgp_loglik_gradient: nothing here is
recorded by autograd, and attend and attend_shared warn where an input requires gradients (not under torch.no_grad()).
"""
import importlib.machinery
import importlib.util
import os

import torch

from .gpx import E_STATE, LIB_PATH, GpxError, lib

EXT_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "gpx_torch.so")
_loaded = None


def ext():
    """The extension over libgpx.so (raises if it has not been built: no fallback)."""
    global _loaded
    if _loaded is None:
        lib()
        if not os.path.exists(EXT_PATH):
            raise GpxError(E_STATE, "gpx_torch.so not built beside %s; run `python -c 'import __graft_entry__ as g; g.build()'`" % LIB_PATH)
        loader = importlib.machinery.ExtensionFileLoader("gpx_torch", EXT_PATH)
        m = importlib.util.module_from_spec(importlib.util.spec_from_file_location("gpx_torch", EXT_PATH, loader=loader))
        loader.exec_module(m)
        m.raise_as(GpxError)
        _loaded = m
    return _loaded


def _stream(q):
    device = q.get_device()
    return torch._C._cuda_getCurrentRawStream(device) if device >= 0 else 0


def attend(q, k, v, scale=None, k_len=None, key_mask=None, q_len=None):
    """o [batch, nq, heads, dim] and lse [batch, heads, nq] (float32) of queries q [batch, nq, heads, dim] over k, v
    [batch, nk, heads_kv, dim].  scale: dim ** -0.5 unless given.  k_len, q_len: int32 [batch], entries and queries that count
    (the others' o is zero, lse -inf); key_mask: bool [batch, nk], True where the entry counts."""
    return (_loaded or ext()).attend(q, k, v, scale, k_len, key_mask, q_len, _stream(q))


def attend_backward(d_o, q, k, v, o, lse, scale=None, k_len=None, key_mask=None, q_len=None):
    """dq, dk, dv for the gradient d_o of attend's o; o and lse as attend returned them, the other arguments as it got them.  d_o may be
    of any size (loss scaling): in float16 too only results that float16 does not hold are lost."""
    return (_loaded or ext()).attend_backward(d_o, q, k, v, o, lse, scale, k_len, key_mask, q_len, _stream(q))


def attend_shared(q, k, v, k_own, v_own, own_len=None, scale=None):
    """o and lse (as attend) of a batch over ONE context: q [batch, nq, heads, dim]; k, v [nk, heads_kv, dim], which every query
    sees; k_own, v_own [batch, n_own, heads_kv, dim], of which own_len[b] (int32 [batch]; None: all) exist, the rows of the nq
    queries last: query i sees the own entries j < own_len[b] - (nq - 1 - i).  The context is read once for the whole batch.  There
    is no gradient call for it."""
    return (_loaded or ext()).attend_shared(q, k, v, k_own, v_own, own_len, scale, _stream(q))
