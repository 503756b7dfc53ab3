"""gpx_attend* at the ends of what the calls take: one entry of any row stride."""
import importlib

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def at(gpu):
    return importlib.import_module("gaussian-object-modelling_amd.attend")


def rnd(t, *shape, seed=0, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(TYPES[t])



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
