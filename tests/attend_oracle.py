"""The attention calls from their formulas in 64 bits on the CPU, with elementwise bounds of what rounding may do to the kernels.

u: half a step of the element type (torch.finfo(t).eps / 2), the most a rounding to it is off, relative to the value; e = 2^-24,
the same in fp32.  A sum of n fp32 terms is off by at most n e times the sum of their sizes, whatever the order.

weights   score s_ij: off by (d + 2) e scale sum|q||k| =: scale-part; exponent, exp and maximum add a few e.  With
          x_i = that at the largest sum|q||k| of the row, a weight and the row's sum of weights are each off by a relative
          x_i + 8 e, and by sum length n e; a normalised weight by ew_i = 2 (x_i + 8 e) + n e.
o         weights rounded (u), product summed in fp32, output rounded: u |o| + (u + ew_i + n e) sum_j p |v|
lse       x_i + n e + 8 e |lse|
backward  p from lse: ew_i + 4 e |lse_i|;  dp: (d + 2) e sum|do||v|;  D from the ROUNDED o: sum|do| (what o is off) + d e sum|do||o|
          ds rounded (u);  the sums' own n e;  outputs rounded (u).
fp16      a weight or ds below 2^-14 keeps an absolute half step of 2^-25; row sums are at least 1 at the weights' scale.
underflow the matrix cores and v_exp_f32 may take fp32 numbers below F = 2^-126 for zero: a weight is off by F besides, so o by
          F sum|v|, dv by F sum|do|, ds by F (|dp| + |D| + 1), and every product and sum by F of its own.
"""
import math

import torch

E = 2.0 ** -24
F = 2.0 ** -126


def half_step(t):
    return 0.0 if t == torch.float32 else torch.finfo(t).eps / 2


def _out_step(t):
    return torch.finfo(t).eps / 2


def _tiny(t):
    return 2.0 ** -25 if t == torch.float16 else F


def forward(q, k, v, scale, seen, t):
    """One head: q [n, d], k, v [m, d], seen [n, m]; fp64.  o, lse, their bounds, and what the backward formulas need."""
    n, d = q.shape
    m = k.shape[0]
    o, lse = torch.zeros(n, d, dtype=torch.float64), torch.full((n,), -math.inf, dtype=torch.float64)
    p = torch.zeros(n, m, dtype=torch.float64)
    some = seen.any(1) if m else torch.zeros(n, dtype=torch.bool)
    k, v = torch.where(seen.any(0)[:, None], k, 0.0), torch.where(seen.any(0)[:, None], v, 0.0)
    q = torch.where(some[:, None], q, 0.0)
    if some.any():
        s = torch.where(seen, scale * (q @ k.T), -math.inf)
        top = s.amax(1, keepdim=True)
        w = torch.where(some[:, None], torch.exp(s - torch.where(some[:, None], top, 0.0)), 0.0)
        total = w.sum(1, keepdim=True)
        p = torch.where(some[:, None], w / torch.where(some[:, None], total, 1.0), 0.0)
        o = p @ v
        lse = torch.where(some, top[:, 0] + torch.log(torch.where(some, total[:, 0], 1.0)), lse)
    u = half_step(t)
    x = torch.zeros(n, dtype=torch.float64)
    if m and n:
        x = ((d + 2) * E * scale * (q.abs() @ k.abs().T) * seen).amax(1)
    ew = 2 * (x + 8 * E) + m * E
    size = p @ v.abs()
    bo = _out_step(t) * o.abs() + (1.01 * u + ew + m * E)[:, None] * size + _tiny(t) * (v.abs().sum(0)[None, :] + 1) + m * F
    bl = x + m * E + 8 * E * (torch.where(some, lse, 0.0).abs() + 1)
    return o, lse, bo, bl, p, ew


def backward(do, q, k, v, scale, seen, t, fwd):
    """One head's dq, dk, dv (fp64) and their bounds."""
    o, lse, bo, _, p, ew = fwd
    n, d = q.shape
    m = k.shape[0]
    some = seen.any(1) if m else torch.zeros(n, dtype=torch.bool)
    used = seen.any(0)
    k, v = torch.where(used[:, None], k, 0.0), torch.where(used[:, None], v, 0.0)
    q, do = torch.where(some[:, None], q, 0.0), torch.where(some[:, None], do, 0.0)
    u, y = half_step(t), _out_step(t)
    dp, D = do @ v.T, (do * o).sum(1, keepdim=True)
    ds = p * (dp - D)
    dv, dq, dk = p.T @ do, scale * (ds @ k), scale * (ds.T @ q)
    ep = (ew + 4 * E * torch.where(some, lse, 0.0).abs())[:, None]
    edp = (d + 2) * E * (do.abs() @ v.abs().T) + (do.abs() * bo).sum(1, keepdim=True) + 2 * d * E * (do.abs() * o.abs()).sum(1, keepdim=True)
    eds = (1.01 * u + 2 * ep + 4 * E) * ds.abs() + 1.01 * p * edp + F * (dp.abs() + D.abs() + 1)
    bv = y * dv.abs() + ((1.01 * u + 2 * ep + n * E) * p).T @ do.abs() + _tiny(t) * (do.abs().sum(0) + 1) + n * F
    bq = y * dq.abs() + scale * ((eds + m * E * ds.abs()) @ k.abs() + _tiny(t) * k.abs().sum(0)) + _tiny(t) + m * F
    bk = y * dk.abs() + scale * ((eds + n * E * ds.abs()).T @ q.abs() + _tiny(t) * q.abs().sum(0)) + _tiny(t) + n * F
    return (dq, dk, dv), (bq, bk, bv)


def seen_of(b, nq, nk, k_len=None, key_mask=None, q_len=None):
    """[b, nq, nk]: which entries a query's softmax is over."""
    s = torch.ones(b, nq, nk, dtype=torch.bool)
    if k_len is not None:
        s &= (torch.arange(nk)[None] < k_len[:, None])[:, None]
    if key_mask is not None:
        s &= key_mask[:, None].bool()
    if q_len is not None:
        s &= (torch.arange(nq)[None] < q_len[:, None])[:, :, None]
    return s


def attend(q, k, v, scale, seen, do=None):
    """Batched, [b, n, h, d] of the element type -> dict name -> (value, bound), fp64."""
    t, (b, nq, hq, d), (nk, hk) = q.dtype, q.shape, k.shape[1:3]
    q, k, v = q.double(), k.double(), v.double()
    out = {"o": (torch.zeros_like(q), torch.zeros_like(q)), "lse": (torch.zeros(b, hq, nq).double(), torch.zeros(b, hq, nq).double())}
    if do is not None:
        do = do.double()
        out.update(dq=(torch.zeros_like(q), torch.zeros_like(q)), dk=(torch.zeros_like(k), torch.zeros_like(k)),
                   dv=(torch.zeros_like(v), torch.zeros_like(v)))
    for i in range(b):
        for h in range(hq):
            g = h // (hq // hk)
            f = forward(q[i, :, h], k[i, :, g], v[i, :, g], scale, seen[i], t)
            out["o"][0][i, :, h], out["o"][1][i, :, h] = f[0], f[2]
            out["lse"][0][i, h], out["lse"][1][i, h] = f[1], f[3]
            if do is not None:
                gr, bd = backward(do[i, :, h], q[i, :, h], k[i, :, g], v[i, :, g], scale, seen[i], t, f)
                for name, at, x, y in zip(("dq", "dk", "dv"), (h, g, g), gr, bd):
                    out[name][0][i, :, at] += x
                    # heads of a group are summed before the one rounding: the sum of the heads' bounds covers it, with
                    # nq more terms in 32 bits for every head
                    out[name][1][i, :, at] += y if name == "dq" else y * (1 + hq // hk * nq * E)
    return out


def shared(q, k, v, k_own, v_own, own_len, scale):
    """k, v [nk, h, d]; the concatenation of the context and every member's own entries."""
    b, nq = q.shape[:2]
    nk, no = k.shape[0], k_own.shape[1]
    kk = torch.cat([k[None].expand(b, -1, -1, -1), k_own], 1)
    vv = torch.cat([v[None].expand(b, -1, -1, -1), v_own], 1)
    n = torch.full((b,), no) if own_len is None else own_len.clamp(0, no)
    last = n[:, None] - (nq - 1 - torch.arange(nq))[None]
    seen = torch.cat([torch.ones(b, nq, nk, dtype=torch.bool), torch.arange(no)[None, None] < last[..., None]], 2)
    return attend(q, kk, vv, scale, seen)
