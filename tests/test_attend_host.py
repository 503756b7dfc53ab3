"""CPU suite of the attention calls: what the C entry points and the torch front refuse, and the oracle's own checks."""
import ctypes as C
import importlib
import math
import struct

import pytest

import attend_oracle as ora

torch = pytest.importorskip("torch")


class Abi:
    """The C entry points, called with the bytes of a gpx_attend_args."""
    FORWARD, BACKWARD, SHARED = range(3)
    _ARGS = struct.Struct("@iiqqqqqqqd" + "Pqqq" * 4 + "PPPPq" + "Pqqq" * 6 + "PPQP")

    def __init__(self, L):
        self.calls = (L.gpx_attend, L.gpx_attend_backward, L.gpx_attend_shared, L.gpx_attend_workspace)

    def _entry(self, i):
        return self.calls[i]


@pytest.fixture(scope="module")
def at(gpx):
    return Abi(gpx.lib())


@pytest.fixture(scope="module")
def front(gpx):
    return importlib.import_module("gaussian-object-modelling_amd.attend")


NAMES = ("scalar device batch nq nk n_own heads heads_kv dim scale q qb qr qh k kb kr kh v vb vr vh o ob orow oh lse q_len k_len "
         "key_mask key_mask_batch d_o gb gr gh dq dqb dqr dqh dk dkb dkr dkh dv dvb dvr dvh k_own kob kor koh v_own vob vor voh own_len "
         "workspace workspace_bytes stream").split()


def args(at, **kv):
    """A call whose pointers are never followed: every one of these is refused before that."""
    d = dict.fromkeys(NAMES, 0)
    d.update(scalar=2, device=-1, batch=2, nq=3, nk=5, heads=4, heads_kv=2, dim=64, scale=0.125)
    for p in ("q", "k", "v", "o", "lse", "d_o", "dq", "dk", "dv", "k_own", "v_own"):
        d[p] = 4096
    for p in NAMES:
        if p in ("qh", "kh", "vh", "oh", "gh", "dqh", "dkh", "dvh", "koh", "voh"):
            d[p] = 64
        if p in ("qr", "kr", "vr", "orow", "gr", "dqr", "dkr", "dvr", "kor", "vor"):
            d[p] = 256
    d.update(kv)
    return at._ARGS.pack(*[d[n] for n in NAMES])


BAD = [(dict(scalar=3), -10), (dict(scalar=-1), -10), (dict(heads=3), -10), (dict(heads=0), -10), (dict(heads_kv=0), -10), (dict(dim=0), -10),
       (dict(dim=12), -10), (dict(dim=136), -10), (dict(batch=-1), -10), (dict(nq=-1), -10), (dict(nk=-1), -10), (dict(n_own=-1), -10),
       (dict(scale=0.0), -10), (dict(scale=-1.0), -10), (dict(scale=math.nan), -10), (dict(scale=math.inf), -10), (dict(scale=1e300), -10),
       (dict(nq=2 ** 31), -10), (dict(nk=2 ** 31), -10), (dict(batch=2 ** 20, nq=2 ** 20), -10), (dict(q=0), -1), (dict(k=0), -1), (dict(v=0), -1),
       (dict(o=0), -1), (dict(lse=0), -1), (dict(q=4098), -10), (dict(kb=3), -10), (dict(vr=4), -10), (dict(qh=-8), -10), (dict(oh=1), -10),
       (dict(kr=0), -10), (dict(vr=56), -10), (dict(kr=2 ** 22 + 8), -10), (dict(qh=2 ** 27), -10), (dict(nq=2 ** 28 + 1), -10), (dict(batch=2 ** 14, nq=2 ** 13, heads=4), -10)]


@pytest.mark.parametrize("kv,code", BAD, ids=lambda x: str(x))
def test_entry_points_refuse(gpx, at, kv, code):
    for call in (at._entry(at.FORWARD), at._entry(at.BACKWARD), at._entry(at.SHARED)):
        assert call(args(at, **kv)) == code
        assert gpx.lib().gpx_last_error()


def test_entry_points_refuse_null(gpx, at):
    for which in range(3):
        assert at._entry(which)(None) == gpx.E_NULL
    n = C.c_size_t(0)
    assert at._entry(3)(None, 0, C.byref(n)) == gpx.E_NULL
    assert at._entry(3)(args(at), 7, C.byref(n)) == gpx.E_BAD_ARG
    assert at._entry(3)(args(at), 0, None) == gpx.E_NULL
    assert at._entry(at.BACKWARD)(args(at, dk=0)) == gpx.E_NULL
    assert at._entry(at.BACKWARD)(args(at, d_o=0)) == gpx.E_NULL
    assert at._entry(at.SHARED)(args(at, n_own=4, k_own=0)) == gpx.E_NULL


def test_outputs_do_not_overlap(gpx, at):
    assert at._entry(at.FORWARD)(args(at, oh=0)) == gpx.E_BAD_ARG
    assert at._entry(at.SHARED)(args(at, oh=56)) == gpx.E_BAD_ARG
    for h in ("dqh", "dkh", "dvh"):
        assert at._entry(at.BACKWARD)(args(at, **{h: 56})) == gpx.E_BAD_ARG


def test_masks_that_a_call_does_not_take(gpx, at):
    for kv in (dict(q_len=4096), dict(k_len=4096), dict(key_mask=4096)):
        assert at._entry(at.SHARED)(args(at, **kv)) == gpx.E_BAD_ARG
    assert at._entry(at.FORWARD)(args(at, key_mask=4096, key_mask_batch=-1)) == gpx.E_BAD_ARG


def test_more_workgroups_than_a_grid_holds(gpx, at):
    n = C.c_size_t(0)
    for which in range(3):
        kv = dict(batch=2 ** 24, nq=1, nk=1, n_own=1, heads=1, heads_kv=1)
        assert at._entry(3)(args(at, **kv), which, C.byref(n)) == gpx.E_BAD_ARG
        kv["batch"] = 2 ** 23
        assert at._entry(3)(args(at, **kv), which, C.byref(n)) == gpx.OK


def test_workspace_sizes(gpx, at):
    def need(which, **kv):
        n = C.c_size_t(0)
        assert at._entry(3)(args(at, **kv), which, C.byref(n)) == gpx.OK
        return n.value

    assert need(at.FORWARD, batch=8, nq=4096, nk=4096) == 0  # enough workgroups without cutting the keys
    assert need(at.FORWARD, batch=1, nq=1, nk=65536) > 0
    assert need(at.BACKWARD, batch=16, nq=4096, nk=4096) >= 16 * 4 * 4096 * 8  # two floats a row from one launch to the next
    assert need(at.BACKWARD) == 0  # one launch, nothing cut
    assert need(at.SHARED, n_own=4) > 0
    assert need(at.FORWARD, batch=0) == 0 and need(at.FORWARD, nq=0) == 0 and need(at.FORWARD, nk=0) == 0


def test_no_gpu_no_result(gpx, at):
    if gpx.device_count() > 0:
        pytest.skip("a HIP device is visible")
    assert at._entry(at.FORWARD)(args(at)) == gpx.E_NO_DEVICE


def test_torch_front_refuses(gpx, front):
    z = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t)  # noqa: E731
    q, k = z(2, 3, 4, 64), z(2, 5, 2, 64)
    for call in (lambda: front.attend(q, k, k),                                    # no CPU path
                 lambda: front.attend(q[0], k, k), lambda: front.attend(q, k[0], k), lambda: front.attend(q.double(), k.double(), k.double()),
                 lambda: front.attend(q, z(2, 5, 3, 64), z(2, 5, 3, 64)), lambda: front.attend_shared(q, k, k, k, k),
                 lambda: front.attend_backward(q, q, k, k, q, z(2, 4, 3))):
        with pytest.raises(gpx.GpxError) as e:
            call()
        assert e.value.code == gpx.E_BAD_ARG and e.value.message
    with pytest.raises(TypeError):
        front.attend(q, k, None)


@pytest.mark.parametrize("t,n", [(torch.float32, 300), (torch.float16, 300), (torch.bfloat16, 12)], ids=str)
def test_oracle_sees_one_entry_too_few(t, n):
    """The bounds tell a result that missed one entry: of 300 in fp32 and fp16, and of a dozen in bf16, where the worst case of
    300 roundings of 2^-8 each is more than one entry's share."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(m, 32, generator=g).double() for m in (4, n, n))
    seen = torch.ones(4, n, dtype=torch.bool)
    a = ora.forward(q, k, v, 32 ** -0.5, seen, t)
    less = seen.clone()
    less[:, n // 2] = False
    c = ora.forward(q, k, v, 32 ** -0.5, less, t)
    assert bool(((a[0] - c[0]).abs() > a[2]).any())
    do = torch.randn(4, 32, generator=g).double()
    ga, bd = ora.backward(do, q, k, v, 32 ** -0.5, seen, t, a)
    gc, _ = ora.backward(do, q, k, v, 32 ** -0.5, less, t, c)
    assert bool(((ga[0] - gc[0]).abs() > bd[0]).any())


def test_oracle_gradients_are_autograds():
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(n, 16, generator=g, dtype=torch.float64) for n in (7, 11, 11, 7))
    seen = torch.rand(7, 11, generator=g) > 0.4
    f = ora.forward(q, k, v, 0.25, seen, torch.float32)
    (dq, dk, dv), _ = ora.backward(do, q, k, v, 0.25, seen, torch.float32, f)
    x = [y.clone().requires_grad_() for y in (q, k, v)]
    o = torch.softmax((0.25 * x[0] @ x[1].T).masked_fill(~seen, -math.inf), 1) @ x[2]
    for a, c in zip((dq, dk, dv), torch.autograd.grad(o, x, do)):
        assert torch.allclose(a, c, atol=1e-12)
