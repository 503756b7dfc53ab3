"""gpx_attend, gpx_attend_backward, gpx_attend_shared against their formulas in 64 bits (tests/attend_oracle.py): values and
gradients within elementwise bounds derived there, masks that leave rows and whole batch members empty, anything in masked places,
strides and layouts, streams and graphs."""
import importlib
import math

import pytest

import attend_oracle as ora

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
#        b, nq, nk, hq, hk, d
SHAPES = [(1, 1, 1, 1, 1, 8), (1, 1, 277, 8, 8, 64), (2, 33, 65, 4, 2, 32), (1, 129, 127, 3, 3, 96), (3, 5, 300, 6, 2, 128),
          (2, 64, 64, 8, 1, 80), (1, 7, 2500, 2, 2, 40), (1, 200, 1000, 2, 1, 128), (1, 1, 5000, 4, 1, 128), (2, 31, 1, 2, 2, 16),
          (1, 257, 33, 2, 2, 64), (1, 3, 129, 40, 2, 24)]
MASKS = ["none", "len", "mask", "len+mask+rows"]


@pytest.fixture(scope="module")
def at(gpu):
    return importlib.import_module("gaussian-object-modelling_amd.attend")


def inputs(t, b, nq, nk, hq, hk, d, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(TYPES[t])  # noqa: E731
    return (1.5 * r(b, nq, hq, d)).to(TYPES[t]), r(b, nk, hk, d), r(b, nk, hk, d), r(b, nq, hq, d)


def masks(kind, b, nq, nk, seed):
    g = torch.Generator().manual_seed(seed + 100)
    k_len = key_mask = q_len = None
    if "len" in kind:
        k_len = torch.randint(0, nk + 1, (b,), generator=g, dtype=torch.int32)
        k_len[0] = max(1, nk - 1)
        if b > 1:
            k_len[-1] = 0
    if "mask" in kind:
        key_mask = torch.rand(b, nk, generator=g) > 0.3
        key_mask[0, 0] = True
        if b > 2:
            key_mask[1] = False
    if "rows" in kind:
        q_len = torch.randint(0, nq + 1, (b,), generator=g, dtype=torch.int32)
        q_len[0] = max(1, nq - 1)
    return dict(k_len=k_len, key_mask=key_mask, q_len=q_len)


def poisoned(x, rows_on):
    """NaN, infinities and the type's lowest value in the rows that do not count ([b, n] bool)."""
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(x.dtype).min], dtype=x.dtype)
    fill = bad[torch.arange(x.numel()) % 4].reshape(x.shape)
    return torch.where(rows_on[:, :, None, None], x, fill)


def cuda(x):
    return None if x is None else x.cuda()


def hold(name, got, want, bound):
    got = got.double().cpu()
    assert got.shape == want.shape, name
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), name
    off = ((got - want).abs() / bound)[~inf]
    assert not torch.isnan(off).any(), name
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 1.0, "%s: %.3g of what rounding explains" % (name, worst)


def both(at, t, shape, kind, seed, scale=None):
    b, nq, nk, hq, hk, d = shape
    q, k, v, do = inputs(t, *shape, seed)
    mk = masks(kind, b, nq, nk, seed)
    seen = ora.seen_of(b, nq, nk, **mk)
    on = seen_keys(b, nk, mk)
    k, v = poisoned(k, on), poisoned(v, on)
    if mk["q_len"] is not None:
        rows = torch.arange(nq)[None] < mk["q_len"][:, None]
        q, do = poisoned(q, rows), poisoned(do, rows)
    want = ora.attend(q, k, v, scale or d ** -0.5, seen, do)
    gm = {n: cuda(x) for n, x in mk.items()}
    gq, gk, gv, gdo = (x.cuda() for x in (q, k, v, do))
    o, lse = at.attend(gq, gk, gv, scale=scale, **gm)
    dq, dk, dv = at.attend_backward(gdo, gq, gk, gv, o, lse, scale=scale, **gm)
    return want, dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv)


def seen_keys(b, nk, mk):
    return ora.seen_of(b, 1, nk, mk["k_len"], mk["key_mask"])[:, 0]


@pytest.mark.parametrize("kind", MASKS)
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_values_and_gradients(at, t, shape, kind):
    want, got = both(at, t, shape, kind, 3)
    for name in got:
        hold(name, got[name], *want[name])


@pytest.mark.parametrize("t", list(TYPES))
def test_every_length_round_a_tile(at, t):
    for nk in (31, 32, 33, 63, 64, 65, 95, 127, 128, 129, 191, 255, 256, 257):
        for nq in (1, 32, 33, 65):
            want, got = both(at, t, (1, nq, nk, 1, 1, 32), "none", nk + nq)
            for name in got:
                hold("%s at %d x %d" % (name, nq, nk), got[name], *want[name])


@pytest.mark.parametrize("t", list(TYPES))
def test_rows_split_over_workgroups_in_the_gradient_of_few_keys(at, t):
    """Few keys and many rows: dK, dV are summed over pieces of the rows; few rows and many keys: dQ over pieces of the keys."""
    for shape in ((1, 1500, 20, 4, 1, 64), (1, 9, 4000, 2, 1, 64)):
        want, got = both(at, t, shape, "mask", 5)
        for name in got:
            hold(name, got[name], *want[name])


# enough (batch, head) pairs to fill the card: workgroups of 64 and of 128 rows, in several orders over the XCDs
WIDE = [(16, 40, 97, 16, 16, 32), (16, 70, 97, 16, 16, 64), (16, 40, 97, 16, 16, 72), (17, 70, 65, 16, 16, 96), (16, 40, 130, 16, 16, 128),
        (19, 70, 130, 14, 14, 120), (2, 100, 150, 8, 4, 64)]


@pytest.mark.parametrize("kind", ["none", "len+mask+rows"])
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("shape", WIDE, ids=lambda s: "x".join(map(str, s)))
def test_many_heads(at, t, shape, kind):
    want, got = both(at, t, shape, kind, 7)
    for name in got:
        hold(name, got[name], *want[name])


@pytest.mark.parametrize("h,d", [(4, 32), (8, 32), (8, 64)])
@pytest.mark.parametrize("t", list(TYPES))
def test_ragged_batch_of_many_workgroups(at, t, h, d):
    """More workgroups than run at once: the batch entries are taken in the order of their lengths (ties, zeros and all), the
    gradients are two launches."""
    b, nq, nk, hq, hk = 24, 1100, 150, h, h
    q, k, v, do = inputs(t, b, nq, nk, hq, hk, d, 13)
    n = torch.randint(0, nk + 1, (b,), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    n[3] = n[4] = n[11] = 77
    n[0] = n[23] = 0
    want = ora.attend(q, k, v, d ** -0.5, ora.seen_of(b, nq, nk, n), do)
    g = [x.cuda() for x in (q, k, v, do)]
    o, lse = at.attend(*g[:3], k_len=n.cuda())
    got = dict(zip(("dq", "dk", "dv"), at.attend_backward(g[3], *g[:3], o, lse, k_len=n.cuda())), o=o, lse=lse)
    for name in got:
        hold(name, got[name], *want[name])


def test_refusals(gpu, at):
    q, k, v, do = (x.cuda() for x in inputs("f32", 2, 3, 5, 4, 2, 64, 0))
    o, lse = at.attend(q, k, v)
    n = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    bad = [lambda: at.attend(q, k.half(), v), lambda: at.attend(q, k.cpu(), v), lambda: at.attend(q, k, v[:, :4]), lambda: at.attend(q, k, v[..., :32]),
           lambda: at.attend(q[..., :60], k[..., :60], v[..., :60]), lambda: at.attend(q, k, v, scale=0.0), lambda: at.attend(q, k, v, scale=math.nan), lambda: at.attend(q, k, v, scale=math.inf),
           lambda: at.attend(q, k, v, k_len=n.long()), lambda: at.attend(q, k, v, k_len=n[:1]), lambda: at.attend(q, k, v, k_len=n.cpu()),
           lambda: at.attend(q, k, v, q_len=n[None]), lambda: at.attend(q, k, v, key_mask=torch.ones(2, 4, dtype=torch.bool, device="cuda")),
           lambda: at.attend(q, k, v, key_mask=torch.ones(2, 5, device="cuda")),
           lambda: at.attend(q, k, v, key_mask=torch.ones(2, 10, dtype=torch.bool, device="cuda")[:, ::2]),
           lambda: at.attend(q[:, :, :3], k, v), lambda: at.attend(q, k[:, :, :0], v[:, :, :0]), lambda: at.attend(q.double(), k.double(), v.double()),
           lambda: at.attend_backward(do, q, k, v, o, lse.half()), lambda: at.attend_backward(do, q, k, v, o, lse[:, :2]),
           lambda: at.attend_backward(do[:1], q, k, v, o, lse), lambda: at.attend_backward(do, q, k, v, o.half(), lse),
           lambda: at.attend_shared(q, k, v, k, v), lambda: at.attend_shared(q, k[0], v[0], k[:, :, :1], v), lambda: at.attend_shared(q, k[0], v[0, :4], k, v),
           lambda: at.attend_shared(q, k[0], v[0], k, v, n[:1])]
    for i, call in enumerate(bad):
        with pytest.raises(gpu.GpxError) as e:
            call()
        assert e.value.code in (gpu.E_BAD_ARG, gpu.E_SIZE_MISMATCH), i
    o2, lse2 = at.attend(q, k, v)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_inputs_that_require_gradients(at):
    """Nothing is recorded, views and copies included."""
    q, k, v, _ = (x.cuda().requires_grad_() for x in inputs("f32", 2, 3, 5, 4, 2, 64, 0))
    o, lse = at.attend(q, k.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2), v)
    o2, _ = at.attend_shared(q, k[0], v[0], k, v)
    assert not o.requires_grad and not lse.requires_grad and not o2.requires_grad


def test_no_entries_and_no_queries(at):
    q = torch.randn(2, 3, 4, 64, device="cuda")
    e = torch.empty(2, 0, 2, 64, device="cuda")
    o, lse = at.attend(q, e, e)
    assert o.shape == q.shape and not o.any() and torch.isinf(lse).all() and (lse < 0).all()
    dq, dk, dv = at.attend_backward(torch.ones_like(q), q, e, e, o, lse)
    assert not dq.any() and dk.shape == e.shape and dv.shape == e.shape
    k = torch.randn(2, 5, 2, 64, device="cuda")
    none = torch.empty(2, 0, 4, 64, device="cuda")
    o, lse = at.attend(none, k, k)
    assert o.shape == none.shape and lse.shape == (2, 4, 0)
    dq, dk, dv = at.attend_backward(none, none, k, k, o, lse)
    assert dq.shape == none.shape and not dk.any() and not dv.any()
    o, lse = at.attend(torch.empty(0, 3, 4, 64, device="cuda"), torch.empty(0, 5, 2, 64, device="cuda"), torch.empty(0, 5, 2, 64, device="cuda"))
    assert o.shape == (0, 3, 4, 64)


@pytest.mark.parametrize("t", list(TYPES))
def test_lengths_outside_the_tensor_are_clamped(at, t):
    q, k, v, _ = inputs(t, 3, 4, 40, 2, 2, 32, 1)
    n = torch.tensor([-5, 1000, 2 ** 31 - 1], dtype=torch.int32)
    want = ora.attend(q, k, v, 32 ** -0.5, ora.seen_of(3, 4, 40, n.clamp(0, 40)))
    o, lse = at.attend(q.cuda(), k.cuda(), v.cuda(), k_len=n.cuda(), q_len=torch.tensor([9, 9, 9], dtype=torch.int32).cuda())
    hold("o", o, *want["o"])
    hold("lse", lse, *want["lse"])


@pytest.mark.parametrize("t", list(TYPES))
def test_large_scores_and_late_maxima(at, t):
    """Scores of hundreds, the largest last: the running maximum is raised again and again."""
    q, k, v, do = inputs(t, 1, 40, 700, 2, 2, 64, 9)
    k = (k.float() * torch.linspace(0.1, 12, 700)[None, :, None, None]).to(k.dtype)
    want = ora.attend(q, k, v, 1.0, ora.seen_of(1, 40, 700), do)
    g = [x.cuda() for x in (q, k, v, do)]
    o, lse = at.attend(*g[:3], scale=1.0)
    for name, x in zip(("dq", "dk", "dv"), at.attend_backward(g[3], *g[:3], o, lse, scale=1.0)):
        hold(name, x, *want[name])
    hold("o", o, *want["o"])
    hold("lse", lse, *want["lse"])


@pytest.mark.parametrize("t", list(TYPES))
def test_layouts(at, t):
    """Packed q k v, heads first, rows of a wider tensor, an unaligned view, a broadcast context: the same results."""
    b, n, h, d = 2, 70, 4, 64
    q, k, v, do = inputs(t, b, n, n, h, h, d, 4)
    g = [x.cuda() for x in (q, k, v, do)]
    ref = at.attend(*g[:3])
    rgr = at.attend_backward(g[3], *g[:3], *ref)

    def same(x):
        o, lse = at.attend(*x[:3])
        assert torch.equal(o, ref[0]) and torch.equal(lse, ref[1])
        for a, c in zip(at.attend_backward(x[3], *x[:3], o, lse), rgr):
            assert torch.equal(a, c)

    packed = torch.stack(g[:3], 2)
    same([packed[:, :, i] for i in range(3)] + [g[3]])
    same([x.transpose(1, 2).contiguous().transpose(1, 2) for x in g])
    wide = torch.full((b, n, h, 2 * d), math.nan, dtype=g[0].dtype, device="cuda")
    views = []
    for x in g:
        w = wide.clone()
        w[..., d:] = x
        views.append(w[..., d:])
    same(views)
    off = []
    for x in g:
        w = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape)
        w.copy_(x)
        off.append(w)
    same(off)
    off = []
    for x in g:  # on a 16-byte boundary, not a 32-byte one
        w = torch.empty(x.numel() + 16 // x.element_size(), dtype=x.dtype, device="cuda")[16 // x.element_size():].view(x.shape)
        w.copy_(x)
        off.append(w)
    same(off)
    same([x.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2) for x in g])
    one = [x[:1].expand(b, -1, -1, -1) for x in g[1:3]]
    x, y = at.attend(g[0], *one), at.attend(g[0], *[w.contiguous() for w in one])
    assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


def test_mask_rows_of_a_wider_mask(at):
    q, k, v, _ = (x.cuda() for x in inputs("bf16", 2, 5, 50, 2, 2, 32, 4))
    wide = torch.rand(2, 99, device="cuda") > 0.5
    a = at.attend(q, k, v, key_mask=wide[:, 7:57])
    c = at.attend(q, k, v, key_mask=wide[:, 7:57].contiguous())
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


def test_context_beyond_32_bit_offsets(at):
    """Rows 40 000 elements apart: the last entries lie past 2^32 bytes and past 2^31 elements."""
    n, step, d = 60000, 40000, 64
    base = torch.empty(n * step, dtype=torch.float16, device="cuda")
    k = base.as_strided((1, n, 1, d), (n * step, step, d, 1))
    v = base.as_strided((1, n, 1, d), (n * step, step, d, 1), storage_offset=64)
    g = torch.Generator(device="cuda").manual_seed(1)
    k.copy_(torch.randn(1, n, 1, d, device="cuda", generator=g))
    v.copy_(torch.randn(1, n, 1, d, device="cuda", generator=g))
    for nq in (1, 150):
        q = torch.randn(1, nq, 1, d, device="cuda", generator=g).half()
        do = torch.randn(1, nq, 1, d, device="cuda", generator=g).half()
        kc, vc = k.contiguous(), v.contiguous()
        a, c = at.attend(q, k, v), at.attend(q, kc, vc)
        assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])
        for x, y in zip(at.attend_backward(do, q, k, v, *a), at.attend_backward(do, q, kc, vc, *c)):
            assert torch.equal(x, y)


SHARED = [(2, 1, 277, 15, 8, 8, 64), (5, 1, 1000, 40, 8, 2, 128), (3, 4, 600, 9, 6, 2, 80), (17, 5, 2000, 64, 3, 1, 32), (1, 1, 1, 1, 1, 1, 8),
          (40, 1, 300, 130, 4, 4, 96), (2, 7, 0, 20, 2, 1, 64), (2, 3, 50, 0, 2, 2, 64), (40, 1, 2000, 30, 16, 16, 64), (70, 1, 2100, 30, 16, 16, 128),
          (35, 2, 2100, 30, 16, 16, 80), (70, 1, 2100, 257, 16, 16, 32)]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("shape", SHARED, ids=lambda s: "x".join(map(str, s)))
def test_shared(at, t, shape, ragged):
    b, nq, nk, no, hq, hk, d = shape
    q, k2, v2, _ = inputs(t, b, nq, no, hq, hk, d, 11)
    _, k, v, _ = inputs(t, 1, 1, nk, hk, hk, d, 12)
    n = None
    if ragged:
        n = torch.randint(0, no + 1, (b,), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
        n[0] = no + 3  # clamped
        k2, v2 = (poisoned(x, torch.arange(no)[None] < n[:, None]) for x in (k2, v2))
    want = ora.shared(q, k[0], v[0], k2, v2, n, d ** -0.5)
    o, lse = at.attend_shared(q.cuda(), k[0].cuda(), v[0].cuda(), k2.cuda(), v2.cuda(), cuda(n))
    hold("o", o, *want["o"])
    hold("lse", lse, *want["lse"])


def test_shared_equals_attend_over_the_joined_context(at):
    """A run of the calls together: a member's own entries appended row by row give what one call over all of them gives."""
    b, nk, steps, h, d = 3, 500, 6, 4, 64
    q, k2, v2, _ = (x.cuda() for x in inputs("f32", b, steps, steps, h, h, d, 21))
    _, k, v, _ = (x.cuda() for x in inputs("f32", 1, 1, nk, h, h, d, 22))
    n = torch.empty(b, dtype=torch.int32, device="cuda")
    for i in range(steps):
        n.fill_(i + 1)
        o, lse = at.attend_shared(q[:, i:i + 1], k[0], v[0], k2, v2, n)
        kk = torch.cat([k.expand(b, -1, -1, -1), k2[:, :i + 1]], 1)
        vv = torch.cat([v.expand(b, -1, -1, -1), v2[:, :i + 1]], 1)
        o2, lse2 = at.attend(q[:, i:i + 1], kk, vv)
        # both are within 1e-5 of the exact values, which are of the order of one
        assert (o - o2).abs().max() < 2e-5 and (lse - lse2).abs().max() < 2e-5
    o, lse = at.attend_shared(q, k[0], v[0], k2, v2, n)
    assert (o[:, -1:] - o2).abs().max() < 2e-5


@pytest.mark.parametrize("t", list(TYPES))
def test_gradient_against_differences(at, t):
    """<gradient, direction> against the central difference of <dO, o> in 64 bits."""
    b, nq, nk, hq, hk, d = 1, 6, 50, 4, 2, 32
    q, k, v, do = inputs(t, b, nq, nk, hq, hk, d, 31)
    seen, scale, h = ora.seen_of(b, nq, nk), d ** -0.5, 1e-4
    g = [x.cuda() for x in (q, k, v, do)]
    o, lse = at.attend(*g[:3])
    grads = at.attend_backward(g[3], *g[:3], o, lse)
    bounds = ora.attend(q, k, v, scale, seen, do)
    gen = torch.Generator().manual_seed(5)

    def loss(x):
        s = 0.0
        for head in range(hq):
            f = ora.forward(x[0][0, :, head], x[1][0, :, head // 2], x[2][0, :, head // 2], scale, seen[0], torch.float32)
            s += float((f[0] * do[0, :, head].double()).sum())
        return s

    for i, name in enumerate(("dq", "dk", "dv")):
        x = [y.double() for y in (q, k, v)]
        way = torch.randn(x[i].shape, generator=gen, dtype=torch.float64)
        lo, hi = list(x), list(x)
        lo[i], hi[i] = x[i] - h * way, x[i] + h * way
        slope = (loss(hi) - loss(lo)) / (2 * h)
        got = float((grads[i].double().cpu() * way).sum())
        # third derivatives here are below 1e3 (directions of norm ~ 50): h^2 / 6 of them, and 1e-16 |loss| / h
        assert abs(got - slope) <= float((bounds[name][1] * way.abs()).sum()) + 1e3 * h * h + 1e-9, name


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_streams_and_repeatability(at, t):
    """Calls on two side streams at once give the bits of the default stream's."""
    g = [x.cuda() for x in inputs(t, 2, 40, 3000, 4, 2, 64, 8)]
    ref = at.attend(*g[:3])
    rgr = at.attend_backward(g[3], *g[:3], *ref)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                o, lse = at.attend(*g[:3])
                outs.append((o, lse) + at.attend_backward(g[3], *g[:3], o, lse))
    torch.cuda.synchronize()
    for got in outs:
        for a, c in zip(got, ref + rgr):
            assert torch.equal(a, c)


def test_tensors_on_another_device_than_the_current_one(at):
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    x = inputs("bf16", 2, 40, 300, 4, 2, 64, 8)
    a, c = [y.to("cuda:0") for y in x], [y.to("cuda:1") for y in x]
    o, lse = at.attend(*a[:3])
    o1, lse1 = at.attend(*c[:3])
    assert o1.device.index == 1 and torch.cuda.current_device() == 0
    assert torch.equal(o.cpu(), o1.cpu()) and torch.equal(lse.cpu(), lse1.cpu())
    for y, z in zip(at.attend_backward(a[3], *a[:3], o, lse), at.attend_backward(c[3], *c[:3], o1, lse1)):
        assert torch.equal(y.cpu(), z.cpu())


def test_captured_and_replayed(at):
    """Two graphs (a training step, a shared call) replayed in turn on new inputs and lengths, with eager work between."""
    b, nq, nk, no, hq, hk, d = 2, 3, 3000, 50, 4, 2, 64
    q, k, v, do = (x.cuda() for x in inputs("bf16", b, nq, nk, hq, hk, d, 41))
    k2, v2 = (x.cuda() for x in inputs("bf16", b, 1, no, hq, hk, d, 42)[1:3])
    k_len = torch.tensor([nk, 17], dtype=torch.int32, device="cuda")
    n = torch.tensor([no, 5], dtype=torch.int32, device="cuda")

    def step():
        o, lse = at.attend(q, k, v, k_len=k_len)
        return (o, lse) + at.attend_backward(do, q, k, v, o, lse, k_len=k_len)

    def serve():
        return at.attend_shared(q, k[0], v[0], k2, v2, n)

    graphs = []
    for f in (step, serve):
        f()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = f()
        graphs.append((gr, out, f))
    for r in range(4):
        q.copy_(torch.randn(q.shape, device="cuda"))
        k.copy_(torch.randn(k.shape, device="cuda"))
        k_len.copy_(torch.tensor([nk - 700 * r, 17 * r], dtype=torch.int32))
        n.copy_(torch.tensor([no - r, 7 * r], dtype=torch.int32))
        for gr, _, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for _, out, f in graphs:
            for a, c in zip(out, f()):
                assert torch.equal(a, c)


def test_results_of_a_later_call_do_not_touch_an_earlier_ones(at):
    g = [x.cuda() for x in inputs("f16", 1, 3, 4000, 2, 2, 128, 51)]
    a = at.attend(*g[:3])
    keep = a[0].clone(), a[1].clone()
    at.attend(g[0] * 2, g[1], g[2])
    at.attend_shared(g[0], g[1][0], g[2][0], g[1], g[2])
    assert torch.equal(a[0], keep[0]) and torch.equal(a[1], keep[1])


@pytest.mark.parametrize("t", list(TYPES))
def test_any_positive_scale(at, t):
    for scale in (1e-3, 0.3, 4.0):
        want, got = both(at, t, (1, 20, 90, 2, 2, 32), "none", 6, scale=scale)
        for name in got:
            hold(name, got[name], *want[name])
