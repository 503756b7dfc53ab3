// gpx_attend.hip -- host side of gpx_attend, gpx_attend_backward and gpx_attend_shared (include/gpx.h): checks, how the work is
// cut, workspace layout, launches.  Kernels: gpx_attend_kernel.hpp (forward), gpx_attend_grad.hpp (gradients).
//
// Nothing is kept between calls and nothing is allocated: partial sums live in the caller's workspace.
#include <limits>

#include "gpx_attend.hpp"
#include "gpx_overlap.hpp"
#include "gpx_model.hpp"

namespace {

struct DeviceScope {  // the call runs on args->device; the caller's current device is restored
    int before = -1;
    ~DeviceScope()
    {
        if (before >= 0)
            (void)hipSetDevice(before);
    }
    int enter(int dev)
    {
        int cur = -1;
        if (hipGetDevice(&cur) != hipSuccess) {
            (void)hipGetLastError();
            return fail(GPX_E_NO_DEVICE, "no HIP device: libgpx has no CPU path");
        }
        if (dev < 0 || cur == dev)
            return GPX_OK;
        HIPCHK(hipSetDevice(dev));
        before = cur;
        return GPX_OK;
    }
};

constexpr int64_t MOST_ROWS = (int64_t)1 << 28;  // row counts, and rows x heads of a call: byte offsets of their floats stay in 31 bits

int elem_size(const gpx_attend_args &a) { return a.scalar == GPX_F32 ? 4 : 2; }

// strides keep every row of `dim` elements on a 16-byte boundary
constexpr int64_t LONGEST_ROW = (int64_t)1 << 22, LONGEST_GROUP = (int64_t)1 << 27;
int check_view(const gpx_attend_args &a, const gpx_view &v, bool needed, int64_t n_rows, int64_t group, const char *name)
{
    if (!needed)
        return GPX_OK;
    if (!v.p)
        return fail(GPX_E_NULL, std::string("Empty data pointer: ") + name);
    const int64_t m = 16 / elem_size(a);
    if ((uintptr_t)v.p % 16 || v.batch % m || v.row % m || v.head % m)
        return fail(GPX_E_BAD_ARG, std::string(name) + ": base and strides must be multiples of 16 bytes");
    if (v.batch < 0 || v.row < 0 || v.head < 0)
        return fail(GPX_E_BAD_ARG, std::string(name) + ": strides must not be negative");
    // the kernels address one tile of rows (at most 128, and the heads of a group) with 32-bit byte offsets
    if (v.row > LONGEST_ROW || (n_rows > 1 && v.row < a.dim))
        return fail(GPX_E_BAD_ARG, std::string(name) + ": row stride below dim or above 2^22");
    if (v.head > LONGEST_GROUP / std::max<int64_t>(1, group))
        return fail(GPX_E_BAD_ARG, std::string(name) + ": the heads of a group must lie within 2^27 elements");
    return GPX_OK;
}

int check_args(const gpx_attend_args *pa, int which)
{
    if (!pa)
        return fail(GPX_E_NULL, "Empty argument pointer");
    const gpx_attend_args &a = *pa;
    if (which != GPX_ATTEND_FORWARD && which != GPX_ATTEND_BACKWARD && which != GPX_ATTEND_SHARED)
        return fail(GPX_E_BAD_ARG, "unknown attention call");
    if (a.scalar != GPX_F32 && a.scalar != GPX_F16 && a.scalar != GPX_BF16)
        return fail(GPX_E_BAD_ARG, "scalar must be GPX_F32, GPX_F16 or GPX_BF16");
    if (a.heads < 1 || a.heads_kv < 1 || a.heads % a.heads_kv)
        return fail(GPX_E_BAD_ARG, "heads must be a positive multiple of heads_kv");
    if (a.dim < 8 || a.dim > ATTEND_MAX_DIM || a.dim % 8)
        return fail(GPX_E_BAD_ARG, "dim must be a multiple of 8 up to 128");
    if (a.batch < 0 || a.nq < 0 || a.nk < 0 || a.n_own < 0)
        return fail(GPX_E_BAD_ARG, "negative size");
    if (!(a.scale > 0.0) || !std::isfinite(a.scale) || !std::isfinite((float)(a.scale * ATTEND_LOG2E)))
        return fail(GPX_E_BAD_ARG, "scale must be positive and finite");
    if (a.scale < (double)std::numeric_limits<float>::min())  // as a float it would lose bits or be 0, and 0 x -inf of a masked entry is NaN
        return fail(GPX_E_BAD_ARG, "scale must be at least 2^-126");
    if (a.batch > MOST_ROWS || a.nq > MOST_ROWS || a.nk > MOST_ROWS || a.n_own > MOST_ROWS || a.heads > 65536 ||
        a.batch * a.nq > MOST_ROWS || a.batch * a.nq * a.heads > MOST_ROWS ||
        (a.batch > 0 && (std::max(a.nk, a.n_own) / 32 + 1) * a.heads_kv > MOST_ROWS / a.batch))
        return fail(GPX_E_BAD_ARG, "too many rows for one call");
    return GPX_OK;
}

int check_data(const gpx_attend_args &a, int which)
{
    const bool rows = a.batch > 0 && a.nq > 0, keys = a.batch > 0 && a.nk > 0, own = a.batch > 0 && a.n_own > 0;
    int rc;
    const int64_t G = a.heads / a.heads_kv;
    // an output's rows and heads are written by different workgroups
#define OUTPUT(V_, ON_, N_, H_)                                                                           \
    if ((rc = check_view(a, a.V_, ON_, N_, 1, #V_)) != GPX_OK)                                            \
        return rc;                                                                                        \
    if ((ON_) && (H_) > 1 && a.V_.head < a.dim)                                                           \
    return fail(GPX_E_BAD_ARG, #V_ ": the heads of an output must not overlap")
#define VIEW(V_, ON_, N_, G_)                                 \
    if ((rc = check_view(a, a.V_, ON_, N_, G_, #V_)) != GPX_OK) \
    return rc
    VIEW(q, rows, a.nq, G);
    VIEW(k, keys, a.nk, 1);
    VIEW(v, keys, a.nk, 1);
    if (which == GPX_ATTEND_BACKWARD) {
        VIEW(o, rows, a.nq, G);
    } else {
        OUTPUT(o, rows, a.nq, a.heads);
    }
    if (rows && !a.lse)
        return fail(GPX_E_NULL, "Empty data pointer: lse");
    if (which == GPX_ATTEND_SHARED) {
        VIEW(k_own, own, a.n_own, 1);
        VIEW(v_own, own, a.n_own, 1);
    }
    if (which == GPX_ATTEND_BACKWARD) {
        VIEW(d_o, rows, a.nq, G);
        OUTPUT(dq, rows, a.nq, a.heads);
        OUTPUT(dk, keys, a.nk, a.heads_kv);
        OUTPUT(dv, keys, a.nk, a.heads_kv);
    }
#undef VIEW
#undef OUTPUT
    if (a.key_mask && a.key_mask_batch < 0)
        return fail(GPX_E_BAD_ARG, "key_mask_batch must not be negative");
    if (which == GPX_ATTEND_SHARED && (a.q_len || a.k_len || a.key_mask))
        return fail(GPX_E_BAD_ARG, "gpx_attend_shared takes own_len only");
    return GPX_OK;
}

// an output's batch entries, rows and heads are written by different workgroups
int check_outputs(const gpx_attend_args &a, int which)
{
    const bool rows = a.batch > 0 && a.nq > 0, keys = a.batch > 0 && a.nk > 0;
    const auto bad = [&](const gpx_view &v, bool on, int64_t n, int64_t heads) {
        return on && rows_overlap({v.batch, v.row, v.head}, {a.batch, n, heads}, a.dim) != 0;
    };
    const char *name = nullptr;
    if (which != GPX_ATTEND_BACKWARD)
        name = bad(a.o, rows, a.nq, a.heads) ? "o" : nullptr;
    else
        name = bad(a.dq, rows, a.nq, a.heads) ? "dq" : bad(a.dk, keys, a.nk, a.heads_kv) ? "dk" : bad(a.dv, keys, a.nk, a.heads_kv) ? "dv" : nullptr;
    return name ? fail(GPX_E_BAD_ARG, std::string(name) + ": the batch entries, rows and heads of an output must not overlap") : GPX_OK;
}

// `pieces` of [0, n) in whole steps of `step`, of at least `least` steps each: where `blocks` workgroups are less than half
// of what the CUs hold (`per_cu` each), enough pieces to fill them
void cut(int64_t blocks, int64_t n, int step, int least, int cus, int per_cu, int *pieces, int *chunk)
{
    int64_t p = 1;
    const int64_t steps = std::max<int64_t>(1, (n + step - 1) / step);
    if (2 * blocks < (int64_t)cus * per_cu && blocks > 0)
        p = std::min<int64_t>((int64_t)cus * per_cu / blocks, steps / least);
    p = std::max<int64_t>(p, 1);
    const int64_t per = (steps + p - 1) / p;
    *chunk = (int)(per * step);
    *pieces = (int)((steps + per - 1) / per);
}

int64_t blocks_of(int64_t rows, int64_t per) { return (rows + per - 1) / per; }

// Waves along the rows: the more rows share a tile of keys, the less often the keys are read -- as long as the workgroups, times the
// pieces the key range may be cut into, give every CU one; else fewer rows and more of the key range at once.
int waves_for(int esz, int dt, int64_t rows, int64_t groups, int64_t n, int (*step)(int esz, int dt, int wm), int least, int cus)
{
    const int lo = attend_least_wm(esz, dt);
    // 129 .. 192 rows: three workgroups of 64, not two of 128 (6-13 % less on six shapes; fp32 with 96 and 128 features, where a
    // workgroup of 64 rows is alone on its CU, 12 % more)
    int wm = rows <= 32 ? 1 : rows <= 64 || (rows > 128 && rows <= 192 && (esz == 2 || dt <= 2)) ? 2 : 4;
    while (wm > lo && blocks_of(rows, 32 * wm) * groups * std::max<int64_t>(1, n / step(esz, dt, wm) / least) < cus)
        wm /= 2;
    return std::max(wm, lo);
}
int fwd_step(int esz, int dt, int wm) { return attend_fwd_bn(esz, dt, wm); }
int dq_step(int, int, int wm) { return attend_dq_bn(wm); }

struct Plan {
    int wm = 4;                         // waves along the rows
    int splits = 1, chunk = 0;          // forward / the shared context
    int own_splits = 0, own_chunk = 0;  // the own part
    int mtiles = 1, own_mtiles = 1, ktiles = 1;  // workgroups along the rows, along the keys (backward)
    bool fused = false;
    int k_splits = 1, k_chunk = 0;      // backward, dK dV: pieces of the rows
    size_t ml = 0, po = 0, pk = 0, pv = 0, total = 0;  // offsets into the workspace (ml: the row statistics in a backward call)
};

size_t up(size_t x) { return (x + 255) & ~(size_t)255; }

// Pieces are joined by one more launch (4 us), and each writes what it summed: 4 bytes per row and feature where a step of the key range
// reads 2 esz per key.  Not below two steps each, nor (along the rows) below what is written, wm steps.  Two instead of six over
// forty small shapes: 5 % less in the mean, a row over 1400 entries 21.6 -> 13.4 us, 41 queries' training step over 2000 entries
// 55 -> 32 us, the slowest change 74 -> 79 us.
int least_steps(int wm) { return std::max(2, wm); }
constexpr int LEAST_DKV_STEPS = 2;

Plan plan_of(const gpx_attend_args &a, int which, int cus)
{
    Plan p;
    const int64_t G = a.heads / a.heads_kv;
    const int esz = elem_size(a), dt = attend_dt((int)a.dim);
    const size_t rid = (size_t)a.batch * a.nq * a.heads;
    if (which == GPX_ATTEND_SHARED) {
        const int R = (int)(a.batch * a.nq * G), Ro = (int)(a.nq * G);
        const int wm = p.wm = waves_for(esz, dt, R, a.heads_kv, a.nk, fwd_step, 1, cus), wo = attend_least_wm(esz, dt);
        p.mtiles = (int)blocks_of(R, 32 * wm), p.own_mtiles = (int)blocks_of(Ro, 32 * wo);
        if (a.nk > 0)
            // a piece writes 4 bytes a row and feature where its keys are 2 esz: pieces of wm steps keep that below what they read
            cut(p.mtiles * a.heads_kv, a.nk, attend_fwd_bn(esz, dt, wm), wm, cus, attend_fwd_per_cu(esz, dt, wm), &p.splits, &p.chunk);
        else
            p.splits = 0;
        if (a.n_own > 0 || a.nk == 0)
            cut(p.own_mtiles * a.heads_kv * a.batch, a.n_own, attend_fwd_bn(esz, dt, wo), 1, cus, 1, &p.own_splits, &p.own_chunk);
        const size_t slots = p.splits + p.own_splits;
        p.ml = 0;
        p.po = up(slots * rid * sizeof(float2));
        p.total = p.po + slots * rid * a.dim * sizeof(float);
        return p;
    }
    const int R = (int)(a.nq * G);
    const int wm = p.wm = waves_for(esz, dt, R, a.heads_kv * a.batch, a.nk, which == GPX_ATTEND_FORWARD ? fwd_step : dq_step, 2, cus);
    p.mtiles = (int)blocks_of(R, 32 * wm);
    const int64_t blocks = p.mtiles * a.heads_kv * a.batch;
    if (which == GPX_ATTEND_FORWARD) {
        cut(blocks, a.nk, attend_fwd_bn(esz, dt, wm), least_steps(wm), cus, attend_fwd_per_cu(esz, dt, wm), &p.splits, &p.chunk);
        if (p.splits > 1) {
            p.po = up(p.splits * rid * sizeof(float2));
            p.total = p.po + p.splits * rid * a.dim * sizeof(float);
        }
        return p;
    }
    p.ktiles = (int)blocks_of(a.nk, ATTEND_DKV_KEYS);
    cut(blocks, a.nk, attend_dq_bn(wm), least_steps(wm), cus, attend_dq_per_cu(esz, dt, wm), &p.splits, &p.chunk);
    cut(p.ktiles * a.heads_kv * a.batch, R, attend_dkv_br(esz), LEAST_DKV_STEPS, cus, attend_dkv_per_cu(esz, dt), &p.k_splits, &p.k_chunk);
    // One launch for dQ and dK, dV together where all their workgroups run at once, or in two rounds of two and more a CU: two small
    // objects 29 -> 20 us.  (With 96 and 128 features the joint kernel is alone on its CU: four batches of 1232 x 874 took 118 us
    // instead of 97.)
    const int both = attend_both_per_cu(esz, dt, wm);
    p.fused = R > 0 && a.nk > 0 &&
              ((int64_t)p.mtiles * p.splits + (int64_t)p.ktiles * p.k_splits) * a.heads_kv * a.batch <= (int64_t)cus * both * (both > 1 ? 2 : 1);
    size_t at = p.fused ? 0 : up(2 * rid * sizeof(float));
    p.po = at;
    if (p.splits > 1)
        at = up(at + p.splits * rid * a.dim * sizeof(float));
    const size_t kv = (size_t)a.batch * a.nk * a.heads_kv * a.dim * sizeof(float);
    p.pk = at;
    if (p.k_splits > 1)
        at = up(at + p.k_splits * kv);
    p.pv = at;
    if (p.k_splits > 1)
        at = up(at + p.k_splits * kv);
    p.total = at;
    return p;
}

// a grid holds less than 2^32 threads: 2^24 workgroups
bool launches_fit(const gpx_attend_args &a, int which, const Plan &p)
{
    const int64_t most = ((int64_t)1 << 24) - 1, pairs = a.heads_kv * a.batch, rows = a.batch * a.nq * a.heads;
    if (which == GPX_ATTEND_SHARED)
        return (int64_t)p.mtiles * p.splits * a.heads_kv + (int64_t)p.own_mtiles * p.own_splits * pairs <= most && rows / 4 < most;
    if ((int64_t)p.mtiles * p.splits * pairs > most || (p.splits > 1 && rows / 4 >= most))
        return false;
    return which == GPX_ATTEND_FORWARD || (int64_t)p.ktiles * p.k_splits * pairs <= most;
}

int cu_count(const gpx_attend_args &a)
{
    int dev = a.device;
    if (dev < 0)
        dev = device_backend()->get_device();
    const int n = dev < 0 ? 0 : device_cu_count(dev);
    return n > 0 ? n : 256;
}

AttendRows rows_of(const gpx_attend_args &a)
{
    AttendRows r;
    r.q = a.q.p;
    r.qb = a.q.batch, r.qr = a.q.row, r.qh = a.q.head;
    r.len = a.q_len;
    r.M = (int)a.nq;
    r.G = (int)(a.heads / a.heads_kv);
    r.Hk = (int)a.heads_kv;
    r.D = (int)a.dim;
    r.R = r.M * r.G;
    r.grid_b = (int)a.batch;
    r.by_m = DivBy((unsigned)std::max(1, r.M));
    r.by_g = DivBy((unsigned)r.G);
    r.by_hk = DivBy((unsigned)r.Hk);
    return r;
}
void set_grid(AttendFwd &f, int wm, int mtiles, int splits, int chunk)
{
    f.wm = wm, f.mtiles = mtiles, f.splits = splits, f.chunk = chunk;
    f.by_mtiles = DivBy((unsigned)mtiles);
    f.by_splits = DivBy((unsigned)std::max(1, splits));
    f.order = attend_order(mtiles, (long)splits * f.rows.Hk * f.rows.grid_b, f.keys.len || f.rows.len);
}
// The kernels take what is left of a buffer from rows x stride.  The stride of a single row says nothing (a broadcast one is 0): dim
// stands for it.
AttendKeys keys_of(const gpx_attend_args &a, const gpx_view &k, const gpx_view &v, int64_t n, const int32_t *len, const uint8_t *mask, int64_t mask_b)
{
    AttendKeys s;
    s.k = k.p, s.v = v.p;
    s.kb = k.batch, s.kr = n > 1 ? k.row : a.dim, s.kh = k.head;
    s.vb = v.batch, s.vr = n > 1 ? v.row : a.dim, s.vh = v.head;
    s.n = (int)n;
    s.len = len;
    s.mask = mask;
    s.mask_b = mask_b;
    return s;
}

// longest key ranges first: ragged batches of up to 64 with more workgroups than run at once
int sorts(const gpx_attend_args &a, int64_t blocks, int64_t at_once) { return a.k_len && a.batch > 1 && a.batch <= 64 && blocks > at_once; }

template <typename F>
int by_type(const gpx_attend_args &a, F &&f)
{
    switch (a.scalar) {
    case GPX_F32: f(float()); break;
    case GPX_F16: f(_Float16()); break;
    default: f(__bf16()); break;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
        return fail(GPX_E_HIP, hipGetErrorString(e));
    return GPX_OK;
}

int begin(const gpx_attend_args *pa, int which, DeviceScope &scope, Plan *plan)
{
    int rc = check_args(pa, which);
    if (rc == GPX_OK)
        rc = check_data(*pa, which);
    if (rc != GPX_OK)
        return rc;
    rc = scope.enter(pa->device);
    if (rc == GPX_OK)
        rc = check_outputs(*pa, which);
    if (rc != GPX_OK)
        return rc;
    *plan = plan_of(*pa, which, cu_count(*pa));
    if (!launches_fit(*pa, which, *plan))
        return fail(GPX_E_BAD_ARG, "too many rows for one call");
    if (plan->total > pa->workspace_bytes || (plan->total && (!pa->workspace || (uintptr_t)pa->workspace % 256)))
        return fail(GPX_E_SIZE_MISMATCH, "workspace: gpx_attend_workspace bytes on a 256-byte boundary are needed");
    return GPX_OK;
}

}  // namespace

extern "C" int gpx_attend_workspace(const gpx_attend_args *args, int which, size_t *bytes)
{
    if (!bytes)
        return fail(GPX_E_NULL, "Empty data pointer: bytes");
    const int rc = check_args(args, which);
    if (rc != GPX_OK)
        return rc;
    const Plan p = plan_of(*args, which, cu_count(*args));
    if (!launches_fit(*args, which, p))
        return fail(GPX_E_BAD_ARG, "too many rows for one call");
    *bytes = p.total;
    return GPX_OK;
}

extern "C" int gpx_attend(const gpx_attend_args *args)
{
    DeviceScope scope;
    Plan p;
    const int rc = begin(args, GPX_ATTEND_FORWARD, scope, &p);
    if (rc != GPX_OK)
        return rc;
    const gpx_attend_args &a = *args;
    if (a.batch == 0 || a.nq == 0)
        return GPX_OK;
    AttendFwd f;
    f.rows = rows_of(a);
    f.keys = keys_of(a, a.k, a.v, a.nk, a.k_len, a.key_mask, a.key_mask_batch);
    f.c = (float)(a.scale * ATTEND_LOG2E);
    set_grid(f, p.wm, p.mtiles, p.splits, p.chunk);
    f.o = a.o.p, f.ob = a.o.batch, f.orow = a.o.row, f.oh = a.o.head;
    f.lse = a.lse;
    f.keys.sort = sorts(a, f.blocks(), cu_count(a) * attend_fwd_per_cu(elem_size(a), attend_dt((int)a.dim), p.wm));
    f.slot_rows = (long)(a.batch * a.nq * a.heads);
    if (p.splits > 1) {
        f.pml = (float2 *)((char *)a.workspace + p.ml);
        f.po = (float *)((char *)a.workspace + p.po);
    }
    return by_type(a, [&](auto t) {
        using T = decltype(t);
        attend_launch_fwd<T>(f, (hipStream_t)a.stream);
        if (p.splits > 1)
            attend_launch_join<T>({f.po, f.pml, p.splits, f.slot_rows, (int)a.nq, (int)a.heads, (int)a.dim, f.o, f.ob, f.orow, f.oh, f.lse},
                                  (hipStream_t)a.stream);
    });
}

extern "C" int gpx_attend_shared(const gpx_attend_args *args)
{
    DeviceScope scope;
    Plan p;
    const int rc = begin(args, GPX_ATTEND_SHARED, scope, &p);
    if (rc != GPX_OK)
        return rc;
    const gpx_attend_args &a = *args;
    if (a.batch == 0 || a.nq == 0)
        return GPX_OK;
    AttendFwd f;
    f.c = (float)(a.scale * ATTEND_LOG2E);
    f.slot_rows = (long)(a.batch * a.nq * a.heads);
    f.pml = (float2 *)((char *)a.workspace + p.ml);
    f.po = (float *)((char *)a.workspace + p.po);
    // the shared context: the rows of the whole batch are rows of one grid entry; a context or own part of no rows has no
    // workgroups
    AttendPair w{f, f};
    w.first.rows = w.second.rows = rows_of(a);
    w.first.rows.R = (int)(a.batch * a.nq) * w.first.rows.G;
    w.first.rows.grid_b = 1;
    w.first.keys = keys_of(a, a.k, a.v, a.nk, nullptr, nullptr, 0);
    set_grid(w.first, p.wm, p.mtiles, p.splits, p.chunk);
    w.second.keys = keys_of(a, a.k_own, a.v_own, a.n_own, a.own_len, nullptr, 0);
    w.second.tail = 1;
    w.second.slot0 = p.splits;
    set_grid(w.second, attend_least_wm(elem_size(a), attend_dt((int)a.dim)), p.own_mtiles, p.own_splits, p.own_chunk);
    return by_type(a, [&](auto t) {
        using T = decltype(t);
        attend_launch_pair<T>(w, (hipStream_t)a.stream);
        attend_launch_join<T>({f.po, f.pml, p.splits + p.own_splits, f.slot_rows, (int)a.nq, (int)a.heads, (int)a.dim, a.o.p, a.o.batch,
                               a.o.row, a.o.head, a.lse},
                              (hipStream_t)a.stream);
    });
}

extern "C" int gpx_attend_backward(const gpx_attend_args *args)
{
    DeviceScope scope;
    Plan p;
    const int rc = begin(args, GPX_ATTEND_BACKWARD, scope, &p);
    if (rc != GPX_OK)
        return rc;
    const gpx_attend_args &a = *args;
    if (a.batch == 0)
        return GPX_OK;
    AttendBwd b;
    b.rows = rows_of(a);
    b.keys = keys_of(a, a.k, a.v, a.nk, a.k_len, a.key_mask, a.key_mask_batch);
    b.c = (float)(a.scale * ATTEND_LOG2E);
    b.scale = (float)a.scale;
    b.o = a.o.p, b.ob = a.o.batch, b.orow = a.o.row, b.oh = a.o.head;
    b.dout = a.d_o.p, b.gb = a.d_o.batch, b.gr = a.d_o.row, b.gh = a.d_o.head;
    b.lse = a.lse;
    b.stat = (float *)((char *)a.workspace + p.ml);
    b.wm = p.wm, b.mtiles = p.mtiles, b.ktiles = p.ktiles;
    b.by_mtiles = DivBy((unsigned)std::max(1, p.mtiles));
    b.by_ktiles = DivBy((unsigned)std::max(1, p.ktiles));
    b.q_order = attend_order(p.mtiles, (long)p.splits * b.rows.Hk * b.rows.grid_b, a.k_len || a.q_len);
    b.k_order = attend_order(p.ktiles, (long)p.k_splits * b.rows.Hk * b.rows.grid_b, a.k_len || a.q_len);
    b.by_q_splits = DivBy((unsigned)p.splits);
    b.by_k_splits = DivBy((unsigned)p.k_splits);
    b.dq = a.dq.p, b.dqb = a.dq.batch, b.dqr = a.dq.row, b.dqh = a.dq.head;
    b.dk = a.dk.p, b.dkb = a.dk.batch, b.dkr = a.dk.row, b.dkh = a.dk.head;
    b.dv = a.dv.p, b.dvb = a.dv.batch, b.dvr = a.dv.row, b.dvh = a.dv.head;
    b.keys.sort = sorts(a, (int64_t)p.mtiles * p.splits * a.heads_kv * a.batch, cu_count(a) * attend_dq_per_cu(elem_size(a), attend_dt((int)a.dim), p.wm));
    b.fused = p.fused;
    b.q_splits = p.splits, b.q_chunk = p.chunk;
    b.k_splits = p.k_splits, b.k_chunk = p.k_chunk;
    if (p.splits > 1)
        b.pq = (float *)((char *)a.workspace + p.po);
    if (p.k_splits > 1) {
        b.pk = (float *)((char *)a.workspace + p.pk);
        b.pv = (float *)((char *)a.workspace + p.pv);
    }
    return by_type(a, [&](auto t) { attend_launch_bwd<decltype(t)>(b, (hipStream_t)a.stream); });
}
