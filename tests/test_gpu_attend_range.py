"""gpx_attend* at the ends of what the calls take: one entry of any row stride, weights and dS far below the largest of their row, d_o
of any size, rows without entries that hold NaN, the pieces of fp32 values, scores past the fp32 range.  Bounds: tests/attend_oracle.py,
its absolute terms for GPX_F16 replaced by what the kernels keep (tight)."""
import importlib
import math
import warnings

import pytest

import attend_oracle as ora
from attend_oracle import E, F

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def at(gpu):
    return importlib.import_module("gaussian-object-modelling_amd.attend")


def rnd(t, *shape, seed=0, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(TYPES[t])


def hold(name, got, want, bound):
    got = got.double().cpu()
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), name
    off = ((got - want).abs() / bound)[~inf]
    assert not torch.isnan(off).any(), name
    assert float(off.max()) <= 1.0, "%s: %.3g of what rounding explains" % (name, float(off.max()))


# ---- one entry ---------------------------------------------------------------------------------------------------------------

def one_entry_views(t, b, hk, d, seed):
    """[b, 1, hk, d] views whose row stride is below d."""
    x = rnd(t, b, 1, d, seed=seed).cuda()
    wide = rnd(t, b * hk * d + d, seed=seed + 1).cuda()
    step = 16 // wide.element_size()
    return [x.expand(b, hk, d).unsqueeze(1), x[:, None].expand(b, 7, hk, d)[:, :1], wide.as_strided((b, 1, hk, d), (hk * d, step, d, 1))]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("nq,d", [(1, 64), (40, 128), (300, 24)])
def test_one_entry_of_any_row_stride(at, t, nq, d):
    """With one row its stride means nothing: what a contiguous copy gives, which for a single entry is its values: the weight and the sum are
    the same fp32 number within 2^-22 of one, so 16-bit values come back as they are, fp32 ones within the roundings of six
    products, a reciprocal and its product."""
    b, hq, hk = 3, 4, 2
    q, do = rnd(t, b, nq, hq, d, seed=1).cuda(), rnd(t, b, nq, hq, d, seed=2).cuda()
    for k, v in zip(one_entry_views(t, b, hk, d, 3), one_entry_views(t, b, hk, d, 5)):
        assert k.stride(1) < d and v.stride(1) < d
        kc, vc = k.contiguous(), v.contiguous()
        o, lse = at.attend(q, k, v)
        oc, lc = at.attend(q, kc, vc)
        want = vc.repeat_interleave(hq // hk, 2).expand(b, nq, hq, d)
        assert bool(((o - want).abs() <= 8 * 2.0 ** -24 * want.abs()).all()) if t == "f32" else torch.equal(o, want)
        assert torch.equal(o, oc) and torch.equal(lse, lc)
        for x, y in zip(at.attend_backward(do, q, k, v, o, lse), at.attend_backward(do, q, kc, vc, oc, lc)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("t", list(TYPES))
def test_one_entry_of_any_row_stride_shared(at, t):
    b, nq, hq, hk, d = 3, 2, 4, 2, 64
    q = rnd(t, b, nq, hq, d, seed=1).cuda()
    ctx, own = rnd(t, 1, 70, hk, d, seed=7).cuda()[0], rnd(t, b, 9, hk, d, seed=8).cuda()
    for k, v in zip(one_entry_views(t, b, hk, d, 3), one_entry_views(t, b, hk, d, 5)):
        for args in ((k[0], v[0], own, own), (ctx, ctx, k, v), (k[1], v[1], k, v)):
            x, y = at.attend_shared(q, *args), at.attend_shared(q, *[a.contiguous() for a in args])
            assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


# ---- weights far below the largest ---------------------------------------------------------------------------------------------

def tight(t, q, k, v, scale, do=None):
    """One head (fp64 q [n, d], k, v [m, d]): {name: (value, bound)}.  As attend_oracle's forward and backward, with these absolute
    terms in GPX_F16, which rounds below 2^-14 to multiples of 2^-24 (off by 2^-25): a weight is rounded as 2^7 times its ratio to a
    reference at most the row's largest, so off by 2^-32 of the row's sum; a weight p for dV as 2^12 p: off by 2^-37; a dS
    times a power of two that brings the largest of the row (dQ) or of the entry (dK) to 2^7 and more: off by 2^-32 of that one.  Outputs
    keep the type's own 2^-25."""
    y = torch.finfo(TYPES[t]).eps / 2
    u, f16 = (0.0 if t == "f32" else y), t == "f16"
    out = 2.0 ** -25 if f16 else F
    (n, d), m = q.shape, k.shape[0]
    o, lse, _, bl, p, ew = ora.forward(q, k, v, scale, torch.ones(n, m, dtype=torch.bool), TYPES[t])
    bo = y * o.abs() + (1.01 * u + ew + m * E)[:, None] * (p @ v.abs()) + (2.0 ** -32 if f16 else F) * v.abs().sum(0) + out + m * F
    r = dict(o=(o, bo), lse=(lse, bl))
    if do is None:
        return r
    dp, D = do @ v.T, (do * o).sum(1, keepdim=True)
    ds = p * (dp - D)
    ep = (ew + 4 * E * lse.abs())[:, None]
    edp = (d + 2) * E * (do.abs() @ v.abs().T) + (do.abs() * bo).sum(1, keepdim=True) + 2 * d * E * (do.abs() * o.abs()).sum(1, keepdim=True)
    eds = (1.01 * u + 2 * ep + 4 * E) * ds.abs() + 1.01 * p * edp + F * (dp.abs() + D.abs() + 1)
    far = 1.01 * 2.0 ** -32 if f16 else 0.0
    dv, dq, dk = p.T @ do, scale * (ds @ k), scale * (ds.T @ q)
    r["dv"] = dv, y * dv.abs() + ((1.01 * u + 2 * ep + n * E) * p).T @ do.abs() + (2.0 ** -37 if f16 else F) * do.abs().sum(0) + out + n * F
    r["dq"] = dq, y * dq.abs() + scale * ((eds + m * E * ds.abs() + far * ds.abs().amax(1, keepdim=True)) @ k.abs()) + out + m * F
    r["dk"] = dk, y * dk.abs() + scale * ((eds + n * E * ds.abs() + far * ds.abs().amax(0, keepdim=True)).T @ q.abs()) + out + n * F
    return r


def two_levels(t, n, m, d, below, seed):
    """Every 32nd entry leads, the others' weights are 2^-below of theirs, and the leaders' values are zero: the result is the tail's."""
    q, k, v = (rnd(t, x, d, seed=seed + i, std=s) for i, (x, s) in enumerate(((n, 0.05), (m, 0.05), (m, 1.0))))
    lead = torch.arange(m) % 32 == 0
    q[:, 0] = 1
    k[:, 0] = torch.where(lead, 0.0, -below * math.log(2)).to(k.dtype)
    v = (1000 + 300 * v.float()).to(v.dtype)
    v[lead] = 0
    return q, k, v


def single(at, t, q, k, v, scale, do=None):
    g = [x.cuda()[None, :, None] for x in (q, k, v)]
    o, lse = at.attend(*g, scale=scale)
    got = dict(o=o[0, :, 0], lse=lse[0, 0])
    if do is not None:
        got.update((a, x[0, :, 0]) for a, x in zip(("dq", "dk", "dv"), at.attend_backward(do.cuda()[None, :, None], *g, o, lse, scale=scale)))
    return got


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("below", [10, 14, 17, 20, 22.4, 25.3])
@pytest.mark.parametrize("n,m,d", [(1, 300, 64), (40, 999, 32), (200, 700, 96), (3, 20000, 128)])
def test_tail_far_below_the_leaders(at, t, below, n, m, d):
    q, k, v = two_levels(t, n, m, d, below, 40)
    want = tight(t, q.double(), k.double(), v.double(), 1.0)
    got = single(at, t, q, k, v, 1.0)
    for name in ("o", "lse"):
        hold(name, got[name], *want[name])


@pytest.mark.parametrize("t", list(TYPES))
def test_tail_far_below_the_leaders_shared(at, t):
    for n, m, own in ((2, 900, 70), (1, 5000, 500)):
        q, k, v = two_levels(t, n, m + own, 64, 20, 50)
        want = tight(t, q[-1:].double(), k.double(), v.double(), 1.0)
        o, lse = at.attend_shared(q.cuda()[None, :, None], k[:m, None].cuda(), v[:m, None].cuda(), k[None, m:, None].cuda(), v[None, m:, None].cuda(),
                                  scale=1.0)
        hold("o", o[0, -1:, 0], *want["o"])
        hold("lse", lse[0, 0, -1:], *want["lse"])


def test_long_tail_behind_one_leading_entry(at):
    """131071 entries 20.9 powers of two below the first one, in rows enough that nothing cuts the range."""
    n, m, d = 65536, 131072, 64
    q, k, v = two_levels("f16", 1, m, d, 20.9, 45)
    v[32::32], k[32::32] = v[31::32][:-1], k[31::32][:-1]
    want = tight("f16", q.double(), k.double(), v.double(), 1.0)
    got = single(at, "f16", q.expand(n, d), k, v, 1.0)
    for name in ("o", "lse"):
        for row in (0, 777, n - 1):
            hold(name, got[name][row:row + 1], *want[name])
        assert bool((got[name] == got[name][:1]).all())


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_sum_of_very_many_small_weights(at, t):
    """One leading entry and 2^19 - 1 of 2^-25 of its weight, in rows enough that nothing cuts the range: the sum adds a step's
    weights up before they join it (32 a lane at most), so that (m / 32 + 40) roundings of 2^-24 stand against 2^19 of them."""
    n, m, d = 65536, 2 ** 19, 32
    q = torch.zeros(1, n, 1, d, device="cuda", dtype=TYPES[t])
    k = torch.zeros(1, m, 1, d, device="cuda", dtype=TYPES[t])
    q[..., 0] = 1
    k[:, 1:, :, 0] = -25.0
    scale = math.log(2)
    o, lse = at.attend(q, k, torch.zeros_like(k), scale=scale)
    want = math.log1p((m - 1) * 2.0 ** -25)
    assert (lse.double() - want).abs().max() <= (m / 32 + 40) * E + 1e-6
    assert not o.any()


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("below", [12, 18, 22.4])
@pytest.mark.parametrize("n,m,d", [(64, 300, 64), (33, 999, 32), (200, 700, 96), (2, 9000, 128), (1500, 40, 128)])
def test_gradients_of_a_tail(at, t, below, n, m, d):
    q, k, v = two_levels(t, n, m, d, below, 60)
    v = (v / 512).to(v.dtype)
    do = (rnd(t, n, d, seed=70, std=0.25).float() + 1).to(q.dtype)
    want = tight(t, q.double(), k.double(), v.double(), 1.0, do.double())
    got = single(at, t, q, k, v, 1.0, do)
    for name in got:
        hold(name, got[name], *want[name])


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("size", [1e-6, 1e-4, 1e-3, 1.0, 1e3])
@pytest.mark.parametrize("n,m,d", [(64, 300, 64), (130, 4096, 32), (200, 700, 96), (1024, 257, 128)])
def test_gradients_for_any_size_of_d_o(at, t, size, n, m, d):
    """q and k of a size that brings dK and dQ near one, whatever d_o is: large with a small scale, or small with a large one."""
    grow = 2.0 ** round(math.log2(min(max(size, 2.0 ** -10), 2.0 ** 10)))
    q, k, v, do = (rnd(t, x, d, seed=80 + i, std=s) for i, (x, s) in enumerate(((n, grow), (m, grow), (m, 1.0), (n, size))))
    scale = d ** -0.5 / grow / grow
    # dK, dQ = scale sum dS q: of the order of size / grow.  With q, k grown further apart only one of them is near one
    for x, y in ((q, k), ((q.float() * grow).to(q.dtype), (k.float() / grow).to(k.dtype)), ((q.float() / grow).to(q.dtype), (k.float() * grow).to(k.dtype))):
        if not bool(torch.isfinite(x).all() and torch.isfinite(y).all()):
            continue
        want = tight(t, x.double(), y.double(), v.double(), scale, do.double())
        got = single(at, t, x, y, v, scale, do)
        for name in got:
            hold(name, got[name], *want[name])


def test_gradients_of_large_d_o_in_16_bits(at):
    """dS of some hundred thousand, where scale dS K, scale dS Q and dV fit GPX_F16."""
    n, m, d = 70, 4, 64
    q, k = rnd("f16", n, d, seed=90, std=2e-3), rnd("f16", m, d, seed=91, std=2e-3)
    v, do = rnd("f16", m, d, seed=92, std=100.0), rnd("f16", n, d, seed=93, std=3e3)
    want = tight("f16", q.double(), k.double(), v.double(), 1.0, do.double())
    assert max(float(want[name][0].abs().max()) for name in ("dq", "dk", "dv")) < 60000
    assert float((do.double() @ (v.double() - v.double().mean(0)).T).abs().max()) / m > 2 * 65504
    got = single(at, "f16", q, k, v, 1.0, do)
    for name in got:
        hold(name, got[name], *want[name])


@pytest.mark.parametrize("t", list(TYPES))
def test_gradients_that_grow_along_the_context(at, t):
    """dS grows by many powers of two from the first entries (zero among them) to the last, and falls the other way round."""
    n, m, d = 48, 640, 64
    q, k, v, do = (rnd(t, x, d, seed=100 + i, std=s) for i, (x, s) in enumerate(((n, 0.3), (m, 0.3), (m, 1.0), (n, 1e-3))))
    up = 2.0 ** torch.linspace(-10, 12, m)[:, None]
    up[:70] = 0
    rows = 2.0 ** torch.linspace(-3, 9, n)[:, None]
    for a, c in ((up, rows), (up.flip(0), rows.flip(0))):
        w, g = (v.float() * a).to(v.dtype), (do.float() * c).to(do.dtype)
        want = tight(t, q.double(), k.double(), w.double(), 0.3, g.double())
        got = single(at, t, q, k, w, 0.3, g)
        for name in got:
            hold(name, got[name], *want[name])


# ---- rows that do not count or see nothing, whatever they hold -------------------------------------------------------------------

def bad_values(x):
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(x.dtype).min], dtype=x.dtype)
    return bad[torch.arange(x.numel()) % 4].reshape(x.shape)


EMPTY = [(3, 5, 300, 4, 2, 64), (3, 70, 97, 4, 4, 128), (3, 2, 5000, 2, 1, 96), (3, 600, 40, 4, 1, 32), (24, 1100, 150, 8, 8, 32), (3, 1, 33, 1, 1, 8)]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("shape", EMPTY, ids=lambda s: "x".join(map(str, s)))
def test_masked_out_members_hold_anything(at, t, shape):
    """A member whose mask leaves nothing gives zeros, -inf and zero gradients with NaN and infinities in its q, d_o, k and v, as one of
    length 0 does; the other members' results are those of a call with plain numbers there."""
    b, nq, nk, hq, hk, d = shape
    q, do = rnd(t, b, nq, hq, d, seed=1), rnd(t, b, nq, hq, d, seed=2)
    k, v = rnd(t, b, nk, hk, d, seed=3), rnd(t, b, nk, hk, d, seed=4)
    mask = torch.rand(b, nk, generator=torch.Generator().manual_seed(5)) > 0.3
    mask[0, 0] = mask[2, 0] = True
    mask[1] = False

    def run(*x):
        g = [y.cuda() for y in x]
        o, lse = at.attend(*g[:3], key_mask=mask.cuda())
        return (o, lse) + at.attend_backward(g[3], *g[:3], o, lse, key_mask=mask.cuda())

    plain = run(q, k, v, do)
    for x in (q, k, v, do):
        x[1] = bad_values(x[1])
    got = run(q, k, v, do)
    for x, y, name in zip(got, plain, ("o", "lse", "dq", "dk", "dv")):
        assert torch.equal(x, y), name
    assert not got[0][1].any() and bool((got[1][1] == -math.inf).all()) and not any(x[1].any() for x in got[2:])


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("shape", EMPTY, ids=lambda s: "x".join(map(str, s)))
def test_rows_that_do_not_count_beside_entries_that_are_not_finite(at, t, shape):
    """q_len: o, lse and dq of the rows behind it are zeros and -inf also where an entry that counts is NaN or infinite."""
    b, nq, nk, hq, hk, d = shape
    q, do = rnd(t, b, nq, hq, d, seed=1), rnd(t, b, nq, hq, d, seed=2)
    k, v = rnd(t, b, nk, hk, d, seed=3), rnd(t, b, nk, hk, d, seed=4)
    k[1, nk // 2], v[1, nk // 3] = bad_values(k[1, 0]), bad_values(v[1, 0])
    n = torch.full((b,), nq, dtype=torch.int32)
    n[1] = nq // 2
    g = [x.cuda() for x in (q, k, v, do)]
    o, lse = at.attend(*g[:3], q_len=n.cuda())
    dq, _, _ = at.attend_backward(g[3], *g[:3], o, lse, q_len=n.cuda())
    at_ = nq // 2
    assert not o[1, at_:].any() and bool((lse[1, :, at_:] == -math.inf).all()) and not dq[1, at_:].any()
    assert bool(torch.isnan(o[1, :at_]).any()) or at_ == 0
    for i in (0, 2):
        assert bool(torch.isfinite(o[i]).all() and torch.isfinite(dq[i]).all())


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("nq,nk", [(40, 300), (2, 5000), (200, 90)])
def test_a_row_that_is_not_finite_stays_its_own(at, t, nq, nk):
    """NaN in one query that sees something: NaN in its row of o, lse and dq, the other rows as without it, with a mask and without."""
    q, do = rnd(t, 2, nq, 2, 64, seed=1), rnd(t, 2, nq, 2, 64, seed=2)
    k, v = rnd(t, 2, nk, 2, 64, seed=3), rnd(t, 2, nk, 2, 64, seed=4)
    mask = torch.rand(2, nk, generator=torch.Generator().manual_seed(5)) > 0.3
    mask[:, 0] = True
    row = nq // 2
    for mk in (None, mask.cuda()):
        for what in (math.nan, math.inf):
            bad = q.clone()
            bad[0, row, 1, 5] = what
            a = at.attend(q.cuda(), k.cuda(), v.cuda(), key_mask=mk)
            c = at.attend(bad.cuda(), k.cuda(), v.cuda(), key_mask=mk)
            dq = at.attend_backward(do.cuda(), bad.cuda(), k.cuda(), v.cuda(), *c, key_mask=mk)[0]
            ref = at.attend_backward(do.cuda(), q.cuda(), k.cuda(), v.cuda(), *a, key_mask=mk)[0]
            assert bool(torch.isnan(c[0][0, row, 1]).all()) and bool(torch.isnan(c[1][0, 1, row])) and bool(torch.isnan(dq[0, row, 1]).all())
            for x, y in ((a[0], c[0]), (ref, dq), (a[1].transpose(1, 2), c[1].transpose(1, 2))):
                x, y = x.clone(), y.clone()
                x[0, row, 1] = y[0, row, 1] = 0
                assert torch.equal(x, y)


# ---- fp32 values in pieces -------------------------------------------------------------------------------------------------------

def test_products_of_fp32_values_are_not_biased(at):
    """One product a score, read from lse = ln 2 * x y.  In units of 2^-24 of it: the pieces left out 3.01 (cut off on one side, m < 2^-7 and
    l < 2^-15, rounded on the other, m <= 2^-8 and l <= 2^-17), the addition of the last piece 2 whichever way the matrix core rounds,
    those before it 2^-6 of that, the product with ln 2 1 and ln 2 itself 0.05.  Long runs of ones on both sides, cut off on both, leave
    out 7.8, always towards zero."""
    g = torch.Generator().manual_seed(1)
    x = 1 + torch.rand(4096, generator=g)
    x[:512] = torch.tensor([0x3f80ffff], dtype=torch.int32).view(torch.float32)   # long runs of ones in the lower bits
    x[512:1024] = (torch.randint(0x3f80, 0x3fff, (512,), generator=g, dtype=torch.int32) * 65536 + 0xffff).view(torch.float32)
    x[1024:1536] = (torch.randint(0x3f80, 0x3fff, (512,), generator=g, dtype=torch.int32) * 65536 + 0x7fff).view(torch.float32)
    x[1536:2048] = (torch.randint(0x3f80, 0x3fff, (512,), generator=g, dtype=torch.int32) * 65536 + 0x8080).view(torch.float32)
    y = x[torch.cat([torch.arange(512), 512 + torch.randperm(3584, generator=g)])] * torch.where(torch.rand(4096, generator=g) < 0.5, 1.0, -1.0)
    q, k = torch.zeros(4096, 1, 1, 8), torch.zeros(4096, 1, 1, 8)
    q[:, 0, 0, 3], k[:, 0, 0, 3] = x, y
    _, lse = at.attend(q.cuda(), k.cuda(), torch.zeros_like(k).cuda(), scale=math.log(2))
    want = math.log(2) * x.double() * y.double()
    off = (lse[:, 0, 0].double().cpu() - want) / want.abs()
    assert off.abs().max() <= (3.01 + 2.03 + 1.05) * E


def test_values_of_any_size_in_fp32_come_through(at):
    """Weight one: the pieces of a value add up to it, bit for bit, up to the largest there is."""
    v = torch.randn(64, 1, 2, 64, generator=torch.Generator().manual_seed(2)) * 2.0 ** torch.arange(-90, 38 * 3, 204 / 64)[:64, None, None, None]
    v.clamp_(-3e38, 3e38)
    bits = torch.tensor([0x7f7fffff, 0x7f7f8000, 0x7f7f7fff, 0x7f7f0000, 0x7f7effff, 0x3f80ffff, 0x3fffffff, 0x3f808000, 0x3f818000], dtype=torch.int32)
    v[0, 0, 0, :9] = bits.view(torch.float32)
    v[0, 0, 1, :9] = -bits.view(torch.float32)
    for nk in (1, 40):
        w = torch.full((64, nk, 2, 64), 1.0)
        w[:, :1] = v
        k = torch.zeros_like(w)
        q = torch.ones(64, 3, 2, 64)
        k[:, 1:] = -100.0
        o, _ = at.attend(q.cuda(), k.cuda(), w.cuda(), scale=1.0)
        assert torch.equal(o.cpu(), v.expand(64, 3, 2, 64))


def test_values_in_fp32_that_are_not_finite(at):
    for what in (math.nan, math.inf, -math.inf):
        q, k, v = (rnd("f32", 2, n, 2, 32, seed=i) for i, n in enumerate((5, 70, 70)))
        a = at.attend(q.cuda(), k.cuda(), v.cuda())[0]
        v[0, 33, 1, 7] = what
        o = at.attend(q.cuda(), k.cuda(), v.cuda())[0]
        assert not bool(torch.isfinite(o[0, :, 1, 7]).any())
        o[0, :, 1, 7] = a[0, :, 1, 7]
        assert torch.equal(o, a)


# ---- the smallest scale ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("t", list(TYPES))
def test_smallest_scale(at, t):
    """Equal weights for what counts, none for the rest."""
    q, k, v = (rnd(t, 2, n, 2, 64, seed=i) for i, n in enumerate((40, 75, 75)))
    mask = torch.rand(2, 75, generator=torch.Generator().manual_seed(5)) > 0.3
    mask[:, 0] = True
    want = ora.attend(q, k, v, 2.0 ** -126, ora.seen_of(2, 40, 75, key_mask=mask))
    o, lse = at.attend(q.cuda(), k.cuda(), v.cuda(), scale=2.0 ** -126, key_mask=mask.cuda())
    hold("o", o, *want["o"])
    hold("lse", lse, *want["lse"])


# ---- outputs over themselves -------------------------------------------------------------------------------------------------------

def test_outputs_that_overlap_are_refused(gpu):
    """On the C entry points (attend.py makes its outputs itself): refused before anything is launched, the layouts around them taken."""
    from test_attend_host import Abi, args
    at = Abi(gpu.lib())
    b, n, h, d = 2, 3, 4, 64
    t = {x: torch.zeros(1 << 14, dtype=torch.bfloat16, device="cuda") for x in ("q", "k", "v", "o", "d_o", "dq", "dk", "dv", "k_own", "v_own")}
    lse, work = torch.zeros(b * h * n, device="cuda"), torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    own = {x: y.data_ptr() for x, y in t.items()}
    own.update(lse=lse.data_ptr(), workspace=work.data_ptr(), workspace_bytes=work.numel(), batch=b, nq=n, nk=n, n_own=n, heads=h, heads_kv=h, device=0)
    own.update(ob=768, dqb=768, dkb=768, dvb=768, stream=torch.cuda.current_stream().cuda_stream)
    assert at._entry(at.FORWARD)(args(at, **own)) == gpu.OK and at._entry(at.BACKWARD)(args(at, **own)) == gpu.OK
    assert at._entry(at.SHARED)(args(at, **own)) == gpu.OK
    bad = [(0, 256, 64), (704, 256, 64), (768, 64, 64), (768, 256, 256), (64, 256, 64)]
    for which, names in ((at.FORWARD, ("ob", "orow", "oh")), (at.SHARED, ("ob", "orow", "oh")), (at.BACKWARD, ("dqb", "dqr", "dqh")),
                         (at.BACKWARD, ("dkb", "dkr", "dkh")), (at.BACKWARD, ("dvb", "dvr", "dvh"))):
        for layout in bad:
            assert at._entry(which)(args(at, **{**own, **dict(zip(names, layout))})) == gpu.E_BAD_ARG, (which, names, layout)
        for layout in ((768, 64, 192), (2304, 768, 64), (256, 512, 64)):
            assert at._entry(which)(args(at, **{**own, **dict(zip(names, layout))})) == gpu.OK, (which, names, layout)
    torch.cuda.synchronize()


# ---- scores past the fp32 range ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("nq,nk,first", [(1, 300, 200), (40, 999, 700), (200, 640, 64), (300, 640, 600)])
def test_entries_whose_score_is_below_every_number(at, t, nq, nk, first):
    """Weight zero wherever they lie, also where the first steps of the range hold nothing else."""
    q, v, do = rnd(t, 1, nq, 1, 64, seed=1), rnd(t, 1, nk, 1, 64, seed=2), rnd(t, 1, nq, 1, 64, seed=3)
    k = rnd(t, 1, nk, 1, 64, seed=4)
    q[..., 0], k[..., 0] = 2.0 ** 70, 0.0
    low = k.clone()
    low[:, :first, :, :] = 0
    low[:, :first, :, 0] = -2.0 ** 70
    o, lse = at.attend(q.cuda(), low.cuda(), v.cuda())
    n = nk - first
    want = ora.attend(q, k[:, first:], v[:, first:], 0.125, ora.seen_of(1, nq, n), do)
    # the zeroth feature adds nothing to a score that counts: its size does not enter the bounds
    free = q.clone()
    free[..., 0] = 0
    plain = ora.attend(free, k[:, first:], v[:, first:], 0.125, ora.seen_of(1, nq, n), do)
    assert torch.allclose(plain["o"][0], want["o"][0])
    hold("o", o, plain["o"][0], plain["o"][1])
    hold("lse", lse, plain["lse"][0], plain["lse"][1])
    dq, dk, dv = at.attend_backward(do.cuda(), q.cuda(), low.cuda(), v.cuda(), o, lse)
    hold("dv", dv[:, first:], *plain["dv"])
    assert not dv[:, :first].any() and not dk[:, :first].any()


# ---- gradients that nothing records --------------------------------------------------------------------------------------------------

def test_inputs_that_require_gradients_are_warned_of(at):
    q, k = rnd("f32", 2, 5, 4, 64, seed=1).cuda(), rnd("f32", 2, 9, 4, 64, seed=2).cuda()
    leaf = k.clone().requires_grad_()
    calls = [lambda x: at.attend(q, x, k), lambda x: at.attend(q, k, x), lambda x: at.attend_shared(q, x[0], k[0], k, k), lambda x: at.attend_shared(q, k[0], k[0], k, x)]
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        ref = [call(k) for call in calls]
        with torch.no_grad():
            for call, y in zip(calls, ref):
                assert torch.equal(call(leaf)[0], y[0])
        with pytest.raises(UserWarning):
            calls[0](leaf)
        at.attend_backward(q, q, leaf, k, *at.attend(q, leaf.detach(), k))
    for call, y in zip(calls, ref):
        with pytest.warns(UserWarning, match="attend_backward") as w:
            o, lse = call(leaf)
        assert not o.requires_grad and torch.equal(o, y[0]) and torch.equal(lse, y[1])
        assert w[0].filename == __file__
    with torch.autograd.forward_ad.dual_level():
        with pytest.warns(UserWarning):
            at.attend(torch.autograd.forward_ad.make_dual(q, torch.ones_like(q)), k, k)
