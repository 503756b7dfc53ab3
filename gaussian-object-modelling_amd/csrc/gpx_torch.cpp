// gpx_torch.cpp -- torch tensors in front of gpx_attend, gpx_attend_backward and gpx_attend_shared (include/gpx.h); attend.py documents
// the calls.  Checks, views, output and workspace allocation in C++ because the smallest calls cost little more than that: one
// query over 277 entries took 12.1 us a call with these steps in Python (a kernel launch is 4.5 of them).  No arithmetic here.
#include <torch/extension.h>

#include <cmath>
#include <string>
#include <tuple>

#include "../../include/gpx.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

struct Refused {  // becomes gpx.GpxError(code, message)
    int code;
    std::string msg;
};
[[noreturn]] void refuse(const std::string &msg, int code = GPX_E_BAD_ARG) { throw Refused{code, msg}; }

void check(int rc)
{
    if (rc != GPX_OK)
        throw Refused{rc, gpx_last_error()};
}

std::string shape_of(at::IntArrayRef s)
{
    std::string r = "[";
    for (size_t i = 0; i < s.size(); ++i)
        r += (i ? ", " : "") + std::to_string(s[i]);
    return r + "]";
}

struct Call {
    const bool recording = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;  // nothing here is recorded by autograd
    bool lost = false;        // an input carries derivatives
    gpx_attend_args a{};
    Tensor q;
    int64_t group = 1;
    c10::TensorOptions like;
    Tensor kept[6];  // copies the call reads
    int copies = 0;

    // the checks of q; hk: the key heads
    Call(const Tensor &q_, int64_t hk, std::optional<double> scale) : q(q_)
    {
        if (q.dim() != 4)
            refuse("q must be a [batch, row, head, dim] tensor");
        switch (q.scalar_type()) {
        case at::kFloat: a.scalar = GPX_F32; break;
        case at::kHalf: a.scalar = GPX_F16; break;
        case at::kBFloat16: a.scalar = GPX_BF16; break;
        default: refuse("q must be float32, float16 or bfloat16");
        }
        if (!q.is_cuda())
            refuse("q must be on a GPU: libgpx has no CPU path");
        a.device = q.get_device();
        a.batch = q.size(0), a.nq = q.size(1), a.heads = q.size(2), a.dim = q.size(3), a.heads_kv = hk;
        if (hk < 1 || a.heads < 1 || a.heads % hk)
            refuse("the key heads must divide the query heads");
        if (a.dim < 8 || a.dim > 128 || a.dim % 8)
            refuse("dim must be a multiple of 8 up to 128");
        group = a.heads / hk;
        a.scale = scale ? *scale : 1.0 / std::sqrt((double)a.dim);
        like = q.options();
    }

    // an input's view; a copy of it where the kernels cannot address it (gpx_view in include/gpx.h)
    gpx_view in(const Tensor &x, const char *name, at::IntArrayRef shape, int64_t heads_of_group = 1)
    {
        lost = lost || x.requires_grad() || (x.unsafeGetTensorImpl()->autograd_meta() && x._fw_grad(0).defined());
        if (x.scalar_type() != q.scalar_type() || x.device() != q.device())
            refuse(std::string(name) + " must be a tensor of the type and device of q");
        if (x.sizes() != shape)
            refuse(std::string(name) + " must be of shape " + shape_of(shape) + ", not " + shape_of(x.sizes()), GPX_E_SIZE_MISMATCH);
        const int64_t esz = x.element_size(), b = x.stride(0), r = x.stride(1), h = x.stride(2);
        const bool usable = !(((uint64_t)x.data_ptr() | (uint64_t)((b | r | h) * esz)) & 15) && x.stride(3) == 1 && r <= (int64_t)1 << 22 &&
                            h * heads_of_group <= (int64_t)1 << 27 && (r >= shape[3] || shape[1] <= 1);
        if (usable || x.numel() == 0)
            return {x.data_ptr(), b, r, h};
        Tensor &y = kept[copies++];
        y = at::empty(shape, like);
        y.copy_(x);
        return dense(y);
    }
    static gpx_view dense(const Tensor &y) { return {y.data_ptr(), y.size(1) * y.size(2) * y.size(3), y.size(2) * y.size(3), y.size(3)}; }
    Tensor out(at::IntArrayRef shape, gpx_view &v)
    {
        Tensor y = at::empty(shape, like);
        v = dense(y);
        return y;
    }
    const int32_t *lengths(const OptTensor &x, const char *name)
    {
        if (!x)
            return nullptr;
        if (x->scalar_type() != at::kInt || x->dim() != 1 || x->device() != q.device() || !x->is_contiguous())
            refuse(std::string(name) + " must be a contiguous int32 tensor [batch] on the device of q");
        if (x->size(0) != a.batch)
            refuse(std::string(name) + " must have one entry per batch member", GPX_E_SIZE_MISMATCH);
        return x->data_ptr<int32_t>();
    }
    void mask(const OptTensor &x)
    {
        if (!x)
            return;
        if ((x->scalar_type() != at::kBool && x->scalar_type() != at::kByte) || x->dim() != 2 || x->device() != q.device() ||
            (x->numel() && a.nk != 1 && x->stride(1) != 1))
            refuse("key_mask must be a bool tensor [batch, nk] on the device of q, its rows contiguous");
        if (x->size(0) != a.batch || x->size(1) != a.nk)
            refuse("key_mask must be of shape " + shape_of({a.batch, a.nk}) + ", not " + shape_of(x->sizes()), GPX_E_SIZE_MISMATCH);
        a.key_mask = (const uint8_t *)x->data_ptr();
        a.key_mask_batch = x->stride(0);
    }
    // a loss over the results would miss these inputs' share of its gradient without a word
    void warn_of_lost_gradients() const
    {
        if (recording && lost &&
            PyErr_WarnEx(PyExc_UserWarning,
                         "attend: an input requires gradients, but nothing is recorded by autograd: gradients are explicit calls "
                         "(attend_backward); under torch.no_grad() this warning is not given",
                         2) < 0)
            throw py::error_already_set();
    }
    void run(int which, int (*call)(const gpx_attend_args *), uint64_t stream)
    {
        a.stream = (void *)stream;
        size_t need = 0;
        check(gpx_attend_workspace(&a, which, &need));
        Tensor work;
        if (need) {
            work = at::empty({(int64_t)need}, like.dtype(at::kByte));
            a.workspace = work.data_ptr(), a.workspace_bytes = need;
        }
        check(call(&a));
    }
};

int64_t heads_of(const Tensor &k, int64_t dims)
{
    if (k.dim() != dims)
        refuse(dims == 4 ? "keys must be a [batch, row, head, dim] tensor" : "keys must be a [row, head, dim] tensor");
    return k.size(dims - 2);
}

std::tuple<Tensor, Tensor> attend(const Tensor &q, const Tensor &k, const Tensor &v, std::optional<double> scale, const OptTensor &k_len,
                                  const OptTensor &key_mask, const OptTensor &q_len, uint64_t stream)
{
    Call c(q, heads_of(k, 4), scale);
    gpx_attend_args &a = c.a;
    a.nk = k.size(1);
    const int64_t ks[4] = {a.batch, a.nk, a.heads_kv, a.dim};
    a.q = c.in(q, "q", q.sizes(), c.group);
    a.k = c.in(k, "k", ks);
    a.v = c.in(v, "v", ks);
    a.q_len = c.lengths(q_len, "q_len");
    a.k_len = c.lengths(k_len, "k_len");
    c.mask(key_mask);
    Tensor o = c.out(q.sizes(), a.o);
    Tensor lse = at::empty({a.batch, a.heads, a.nq}, c.like.dtype(at::kFloat));
    a.lse = lse.data_ptr<float>();
    c.warn_of_lost_gradients();
    c.run(GPX_ATTEND_FORWARD, gpx_attend, stream);
    return {o, lse};
}

std::tuple<Tensor, Tensor, Tensor> attend_backward(const Tensor &d_o, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &o,
                                                   const Tensor &lse, std::optional<double> scale, const OptTensor &k_len, const OptTensor &key_mask,
                                                   const OptTensor &q_len, uint64_t stream)
{
    Call c(q, heads_of(k, 4), scale);
    gpx_attend_args &a = c.a;
    a.nk = k.size(1);
    const int64_t ks[4] = {a.batch, a.nk, a.heads_kv, a.dim};
    a.q = c.in(q, "q", q.sizes(), c.group);
    a.k = c.in(k, "k", ks);
    a.v = c.in(v, "v", ks);
    a.o = c.in(o, "o", q.sizes(), c.group);
    a.d_o = c.in(d_o, "d_o", q.sizes(), c.group);
    if (lse.scalar_type() != at::kFloat || lse.device() != q.device() || !lse.is_contiguous())
        refuse("lse must be a contiguous float32 tensor on the device of q");
    const int64_t ls[3] = {a.batch, a.heads, a.nq};
    if (lse.sizes() != at::IntArrayRef(ls))
        refuse("lse must be of shape " + shape_of(ls) + ", not " + shape_of(lse.sizes()), GPX_E_SIZE_MISMATCH);
    a.lse = lse.data_ptr<float>();
    a.q_len = c.lengths(q_len, "q_len");
    a.k_len = c.lengths(k_len, "k_len");
    c.mask(key_mask);
    Tensor dq = c.out(q.sizes(), a.dq), dk = c.out(ks, a.dk), dv = c.out(ks, a.dv);
    c.run(GPX_ATTEND_BACKWARD, gpx_attend_backward, stream);
    return {dq, dk, dv};
}

std::tuple<Tensor, Tensor> attend_shared(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &k_own, const Tensor &v_own,
                                         const OptTensor &own_len, std::optional<double> scale, uint64_t stream)
{
    const int64_t hk = heads_of(k, 3);
    if (heads_of(v, 3) != hk || heads_of(k_own, 4) != hk)
        refuse("k, v, k_own and v_own must have the same heads", GPX_E_SIZE_MISMATCH);
    Call c(q, hk, scale);
    gpx_attend_args &a = c.a;
    a.nk = k.size(0), a.n_own = k_own.size(1);
    const int64_t ks[4] = {1, a.nk, hk, a.dim}, os[4] = {a.batch, a.n_own, hk, a.dim};
    a.q = c.in(q, "q", q.sizes(), c.group);
    a.k = c.in(k.unsqueeze(0), "k", ks);
    a.v = c.in(v.unsqueeze(0), "v", ks);
    a.k_own = c.in(k_own, "k_own", os);
    a.v_own = c.in(v_own, "v_own", os);
    a.own_len = c.lengths(own_len, "own_len");
    Tensor o = c.out(q.sizes(), a.o);
    Tensor lse = at::empty({a.batch, a.heads, a.nq}, c.like.dtype(at::kFloat));
    a.lse = lse.data_ptr<float>();
    c.warn_of_lost_gradients();
    c.run(GPX_ATTEND_SHARED, gpx_attend_shared, stream);
    return {o, lse};
}

PyObject *error_class = nullptr;

}  // namespace

PYBIND11_MODULE(gpx_torch, m)
{
    m.def("attend", &attend);
    m.def("attend_backward", &attend_backward);
    m.def("attend_shared", &attend_shared);
    m.def("raise_as", [](py::object cls) {
        Py_XDECREF(error_class);
        error_class = cls.release().ptr();
    });
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p)
                std::rethrow_exception(p);
        } catch (const Refused &r) {
            py::object e = py::reinterpret_steal<py::object>(PyObject_CallFunction(error_class, "is", r.code, r.msg.c_str()));
            if (e)
                PyErr_SetObject(error_class, e.ptr());
        }
    });
}
