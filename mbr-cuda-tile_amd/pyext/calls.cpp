// Native half of the Python binding: the calls a model makes hundreds of times per chunk, from
// torch tensors straight to the C-ABI of libmbrt.so.  Each function checks what its Python
// wrapper (mbrt/__init__.py) documents, reads pointers, sizes and dtypes from the tensors,
// and enqueues on the given stream handle, or on torch's current stream for None.
//
// What it is for: a small kernel runs for 2-4 us, while a call through ctypes took 8.3 us of host
// time (attribute lookups, a ctypes object per argument, a Structure filled element by
// element), so that a chunk's loops of small calls ran at the host's pace.  From here a call
// takes 3.9 us, most of it the launch: the 60 per-band slices and norms of a chunk, 121
// calls, 1009 -> 475 us; the 40 calls of a one-minute song's overlap-add 335 -> 242 us.
//
// Like ctypes' calls, the library is entered without the interpreter lock.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>


#include <vector>

#include "../../include/mbrt.h"

namespace {

PyObject* g_error = nullptr;  // mbrt.MbrtError(function, status, message)

[[noreturn]] void raise(PyObject* type, const char* msg) {
    PyErr_SetString(type, msg);
    throw python_error();
}

const at::Tensor& tensor(PyObject* o) {
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, "mbrt: expected a torch.Tensor");
    return THPVariable_Unpack(o);
}

// An optional tensor argument: undefined for None.
at::Tensor tensor_or_none(PyObject* o) { return o == Py_None ? at::Tensor() : tensor(o); }

int dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return MBRT_F32;
        case at::kHalf: return MBRT_F16;
        case at::kBFloat16: return MBRT_BF16;
        case at::kLong: return MBRT_I64;
        case at::kInt: return MBRT_I32;
        default: break;
    }
    const std::string msg = std::string("mbrt: unsupported dtype torch.") + torch::getTHPDtype(t.scalar_type())->name;
    raise(PyExc_TypeError, msg.c_str());
}
int dtype_or(const at::Tensor& t, int none) { return t.defined() ? dtype_code(t) : none; }

void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void contig(std::initializer_list<const at::Tensor*> ts) {
    for (const at::Tensor* t : ts)
        if (t->defined() && !t->is_contiguous()) raise(PyExc_ValueError, "mbrt: expected a contiguous tensor");
}

int64_t integer(PyObject* o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
int truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v;
}

int64_t floor_div(int64_t a, int64_t b) {
    if (b == 0) raise(PyExc_ZeroDivisionError, "integer division or modulo by zero");
    return a / b;
}

mbrt_stream_t stream(PyObject* o) {
    if (o == Py_None) return c10::hip::getCurrentHIPStream().stream();
    return reinterpret_cast<mbrt_stream_t>(static_cast<uintptr_t>(integer(o)));
}

template <class F>
PyObject* call(const char* name, F f) {
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = f();
    Py_END_ALLOW_THREADS
    if (status != MBRT_OK) {
        PyObject* e = PyObject_CallFunction(g_error, "sis", name, status, mbrt_last_error());
        if (e != nullptr) {
            PyErr_SetObject(g_error, e);
            Py_DECREF(e);
        }
        throw python_error();
    }
    Py_RETURN_NONE;
}

void count(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) raise(PyExc_TypeError, "mbrt: wrong number of arguments to a native call");
}

void check_dims(const at::Tensor& t) {
    if (t.dim() > MBRT_MAX_DIMS) raise(PyExc_IndexError, "invalid index");
}

#define MBRT_PY(fname) PyObject* fname(PyObject*, PyObject* const* a, Py_ssize_t n)

// fill(t, value, stream)
MBRT_PY(fill) {
    HANDLE_TH_ERRORS
    count(n, 3);
    const at::Tensor& t = tensor(a[0]);
    contig({&t});
    const int dt = dtype_code(t);
    void* p = ptr(t);
    const double v = number(a[1]);
    const int64_t ne = t.numel();
    const mbrt_stream_t st = stream(a[2]);
    return call("mbrt_fill", [&] { return mbrt_fill(p, dt, ne, v, st); });
    END_HANDLE_TH_ERRORS
}

// strided_copy(src, dst, stream)
MBRT_PY(strided_copy) {
    HANDLE_TH_ERRORS
    count(n, 3);
    const at::Tensor &src = tensor(a[0]), &dst = tensor(a[1]);
    contig({&dst});
    if (src.sizes() != dst.sizes()) raise(PyExc_ValueError, "strided_copy: shape mismatch");
    check_dims(src);
    mbrt_strided_meta m{};
    m.ndim = (int32_t)src.dim();
    for (int64_t d = 0; d < src.dim(); ++d) {
        m.dst_shape[d] = src.size(d);
        m.src_strides[d] = src.stride(d);
    }
    const int dt = dtype_code(src);
    void *sp = ptr(src), *dp = ptr(dst);
    const mbrt_stream_t st = stream(a[2]);
    return call("mbrt_strided_copy", [&] { return mbrt_strided_copy(sp, dp, dt, &m, st); });
    END_HANDLE_TH_ERRORS
}

// pad(src, out, before (sequence), value, reflect, stream)
MBRT_PY(pad) {
    HANDLE_TH_ERRORS
    count(n, 6);
    const at::Tensor &src = tensor(a[0]), &out = tensor(a[1]);
    contig({&src, &out});
    check_dims(src);
    mbrt_pad_meta m{};
    m.ndim = (int32_t)src.dim();
    for (int64_t d = 0; d < src.dim(); ++d) {
        m.src_shape[d] = src.size(d);
        m.dst_shape[d] = out.size(d);
        PyObject* b = PySequence_GetItem(a[2], d);
        if (b == nullptr) throw python_error();
        const int64_t v = PyLong_AsLongLong(b);
        Py_DECREF(b);
        if (v == -1 && PyErr_Occurred()) throw python_error();
        m.pad_before[d] = v;
    }
    const int dt = dtype_code(src);
    void *sp = ptr(src), *op = ptr(out);
    const mbrt_stream_t st = stream(a[5]);
    if (truth(a[4])) return call("mbrt_pad_reflect", [&] { return mbrt_pad_reflect(sp, op, dt, &m, st); });
    const float value = (float)number(a[3]);
    return call("mbrt_pad_const", [&] { return mbrt_pad_const(sp, op, dt, &m, value, st); });
    END_HANDLE_TH_ERRORS
}

// cat(srcs (sequence), dim, out, stream)
MBRT_PY(cat) {
    HANDLE_TH_ERRORS
    count(n, 4);
    const at::Tensor& out = tensor(a[2]);
    contig({&out});
    THPObjectPtr seq(PySequence_Fast(a[0], "mbrt.cat: expected a sequence of tensors"));
    if (!seq) throw python_error();
    const Py_ssize_t ns = PySequence_Fast_GET_SIZE(seq.get());
    PyObject** items = PySequence_Fast_ITEMS(seq.get());
    for (Py_ssize_t i = 0; i < ns; ++i) contig({&tensor(items[i])});
    if (out.dim() == 0) raise(PyExc_ZeroDivisionError, "integer division or modulo by zero");
    int64_t dim = integer(a[1]) % out.dim();
    if (dim < 0) dim += out.dim();
    int64_t outer = 1, inner = 1, off = 0;
    for (int64_t d = 0; d < dim; ++d) outer *= out.size(d);
    for (int64_t d = dim + 1; d < out.dim(); ++d) inner *= out.size(d);
    std::vector<mbrt_cat_src> srcs((size_t)ns);
    for (Py_ssize_t i = 0; i < ns; ++i) {
        const at::Tensor& s = tensor(items[i]);
        srcs[i] = mbrt_cat_src{ptr(s), s.size(dim), off};
        off += s.size(dim);
    }
    void* op = ptr(out);
    const int64_t total = out.size(dim), bytes = inner * (int64_t)out.element_size();
    const mbrt_stream_t st = stream(a[3]);
    return call("mbrt_cat", [&] { return mbrt_cat(op, srcs.data(), (int)ns, outer, total, bytes, st); });
    END_HANDLE_TH_ERRORS
}

// rms_norm(x, gamma, out, scale, eps, stream)
MBRT_PY(rms_norm) {
    HANDLE_TH_ERRORS
    count(n, 6);
    const at::Tensor &x = tensor(a[0]), &g = tensor(a[1]), &out = tensor(a[2]);
    contig({&x, &g, &out});
    const int64_t dim = x.size(-1);
    const int xd = dtype_code(x), gd = dtype_code(g), od = dtype_code(out);
    const int64_t rows = floor_div(x.numel(), dim);
    void *xp = ptr(x), *gp = ptr(g), *op = ptr(out);
    const float scale = (float)number(a[3]), eps = (float)number(a[4]);
    const mbrt_stream_t st = stream(a[5]);
    return call("mbrt_rms_norm", [&] { return mbrt_rms_norm(xp, xd, gp, gd, op, od, rows, dim, scale, eps, st); });
    END_HANDLE_TH_ERRORS
}

// residual_add_rms_norm(residual, update, gamma, sum_out | None, normed, scale, eps, stream)
MBRT_PY(residual_add_rms_norm) {
    HANDLE_TH_ERRORS
    count(n, 8);
    const at::Tensor &r = tensor(a[0]), &u = tensor(a[1]), &g = tensor(a[2]), &out = tensor(a[4]);
    const at::Tensor sum = tensor_or_none(a[3]);
    contig({&r, &u, &g, &sum, &out});
    const int64_t dim = r.size(-1);
    const int rd = dtype_code(r), gd = dtype_code(g), od = dtype_code(out), sd = dtype_or(sum, rd);
    const int64_t rows = floor_div(r.numel(), dim);
    void *rp = ptr(r), *up = ptr(u), *gp = ptr(g), *sp = ptr(sum), *op = ptr(out);
    const float scale = (float)number(a[5]), eps = (float)number(a[6]);
    const mbrt_stream_t st = stream(a[7]);
    return call("mbrt_residual_add_rms_norm", [&] {
        return mbrt_residual_add_rms_norm(rp, up, rd, gp, gd, sp, sd, op, od, rows, dim, scale, eps, st);
    });
    END_HANDLE_TH_ERRORS
}

// bias_act(x, bias | None, out, act, stream)
MBRT_PY(bias_act) {
    HANDLE_TH_ERRORS
    count(n, 5);
    const at::Tensor &x = tensor(a[0]), &out = tensor(a[2]);
    const at::Tensor bias = tensor_or_none(a[1]);
    contig({&x, &bias, &out});
    const int64_t cols = x.size(-1);
    const int xd = dtype_code(x), bd = dtype_or(bias, MBRT_F32), od = dtype_code(out);
    const int64_t rows = floor_div(x.numel(), cols);
    void *xp = ptr(x), *bp = ptr(bias), *op = ptr(out);
    const int act = (int)integer(a[3]);
    const mbrt_stream_t st = stream(a[4]);
    return call("mbrt_bias_act", [&] { return mbrt_bias_act(xp, xd, bp, bd, op, od, rows, cols, act, st); });
    END_HANDLE_TH_ERRORS
}

// glu(x, out, stream)
MBRT_PY(glu) {
    HANDLE_TH_ERRORS
    count(n, 3);
    const at::Tensor &x = tensor(a[0]), &out = tensor(a[1]);
    contig({&x, &out});
    const int64_t full = x.size(-1);
    if (full % 2 != 0) raise(PyExc_ValueError, "glu_last_dim: last dimension must be even");
    const int xd = dtype_code(x), od = dtype_code(out);
    const int64_t rows = floor_div(x.numel(), full);
    void *xp = ptr(x), *op = ptr(out);
    const mbrt_stream_t st = stream(a[2]);
    return call("mbrt_glu_last_dim", [&] { return mbrt_glu_last_dim(xp, xd, op, od, rows, full / 2, st); });
    END_HANDLE_TH_ERRORS
}

// gate_merge(attn, gate, out, layout, gate_is_logit, stream)
MBRT_PY(gate_merge) {
    HANDLE_TH_ERRORS
    count(n, 6);
    const at::Tensor &at_ = tensor(a[0]), &g = tensor(a[1]), &out = tensor(a[2]);
    contig({&at_, &g, &out});
    const int layout = (int)integer(a[3]);
    if (at_.dim() != 4) raise(PyExc_ValueError, "gate_merge: expected a 4-d attention output");
    const bool bhnd = layout == MBRT_LAYOUT_BHND;
    const int64_t B = at_.size(0), H = at_.size(bhnd ? 1 : 2), N = at_.size(bhnd ? 2 : 1), D = at_.size(3);
    const int ad = dtype_code(at_), gd = dtype_code(g), od = dtype_code(out), logit = truth(a[4]);
    void *ap = ptr(at_), *gp = ptr(g), *op = ptr(out);
    const mbrt_stream_t st = stream(a[5]);
    return call("mbrt_sigmoid_gate_merge", [&] {
        return mbrt_sigmoid_gate_merge(ap, ad, gp, gd, logit, op, od, B, H, N, D, layout, st);
    });
    END_HANDLE_TH_ERRORS
}

// softmax(x, out, scale, stream)
MBRT_PY(softmax) {
    HANDLE_TH_ERRORS
    count(n, 4);
    const at::Tensor &x = tensor(a[0]), &out = tensor(a[1]);
    contig({&x, &out});
    const int64_t cols = x.size(-1);
    const int xd = dtype_code(x), od = dtype_code(out);
    const int64_t rows = floor_div(x.numel(), cols);
    void *xp = ptr(x), *op = ptr(out);
    const float scale = (float)number(a[2]);
    const mbrt_stream_t st = stream(a[3]);
    return call("mbrt_softmax_rows", [&] { return mbrt_softmax_rows(xp, xd, op, od, rows, cols, scale, st); });
    END_HANDLE_TH_ERRORS
}

// split_qkv_rotary(qkv, cos, sin, q, k, v, heads, stream)
MBRT_PY(split_qkv_rotary) {
    HANDLE_TH_ERRORS
    count(n, 8);
    const at::Tensor &qkv = tensor(a[0]), &c = tensor(a[1]), &s = tensor(a[2]), &q = tensor(a[3]), &k = tensor(a[4]),
                     &v = tensor(a[5]);
    contig({&qkv, &c, &s, &q, &k, &v});
    if (qkv.dim() != 3) raise(PyExc_ValueError, "split_qkv_rotary: expected qkv [B, N, 3 H D]");
    const int64_t heads = integer(a[6]), B = qkv.size(0), N = qkv.size(1), D = floor_div(qkv.size(2), 3 * heads);
    const int64_t out_n = q.size(2);
    const int id = dtype_code(qkv), td = dtype_code(c), od = dtype_code(q);
    void *ip = ptr(qkv), *cp = ptr(c), *sp = ptr(s), *qp = ptr(q), *kp = ptr(k), *vp = ptr(v);
    const mbrt_stream_t st = stream(a[7]);
    return call("mbrt_split_qkv_heads_rotary", [&] {
        return mbrt_split_qkv_heads_rotary(ip, id, cp, sp, td, qp, kp, vp, od, B, N, heads, D, out_n, st);
    });
    END_HANDLE_TH_ERRORS
}

// attention_ex(q, k, v, (B, H, n_q, n_k, D), (six strides), cos | None, sin | None, gate | None, gate_is_logit,
//              out, scale, p_precision, stream)
MBRT_PY(attention_ex) {
    HANDLE_TH_ERRORS
    count(n, 13);
    const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]), &out = tensor(a[9]);
    const at::Tensor c = tensor_or_none(a[5]), s = tensor_or_none(a[6]), g = tensor_or_none(a[7]);
    int64_t z[11];
    for (int i = 0; i < 5; ++i) z[i] = integer(PyTuple_GET_ITEM(a[3], i));
    for (int i = 0; i < 6; ++i) z[5 + i] = integer(PyTuple_GET_ITEM(a[4], i));
    const int dt = dtype_code(q), td = dtype_or(c, MBRT_F32), gd = dtype_or(g, MBRT_F32), od = dtype_code(out);
    const int logit = truth(a[8]), pm = (int)integer(a[11]);
    void *qp = ptr(q), *kp = ptr(k), *vp = ptr(v), *cp = ptr(c), *sp = ptr(s), *gp = ptr(g), *op = ptr(out);
    const float scale = (float)number(a[10]);
    const mbrt_stream_t st = stream(a[12]);
    return call("mbrt_attention_ex", [&] {
        return mbrt_attention_ex(qp, kp, vp, dt, z[0], z[1], z[2], z[3], z[4], z[5], z[6], z[7], z[8], z[9], z[10], cp,
                                 sp, td, gp, gd, logit, op, od, scale, pm, st);
    });
    END_HANDLE_TH_ERRORS
}

// A call on the device of these tensors, which becomes the current one where it is not.
class OnDevice {
public:
    explicit OnDevice(std::initializer_list<const at::Tensor*> ts) : dev_((*ts.begin())->device()) {
        for (const at::Tensor* t : ts)
            if (t->defined() && (!t->is_cuda() || t->device() != dev_))
                raise(PyExc_ValueError, "mbrt: expected tensors on one GPU");
        if (dev_.index() != c10::hip::current_device()) guard_.reset_device(dev_);
    }
    mbrt_stream_t stream(PyObject* o) const {
        if (o == Py_None) return c10::hip::getCurrentHIPStream(dev_.index()).stream();
        return reinterpret_cast<mbrt_stream_t>(static_cast<uintptr_t>(integer(o)));
    }

private:
    at::Device dev_;
    c10::OptionalDeviceGuard guard_;
};

void unit_last(std::initializer_list<const at::Tensor*> ts) {
    for (const at::Tensor* t : ts)
        if (t->defined() && t->dim() && t->size(-1) > 1 && t->stride(-1) != 1)
            raise(PyExc_ValueError, "mbrt: expected a contiguous last dim");
}

// Strides that are used, the same in both (those of a single index are not).
bool strided_alike(const at::Tensor& a, const at::Tensor& b) {
    if (a.numel() == 0) return true;
    for (int64_t d = 0; d < a.dim(); ++d)
        if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
    return true;
}

[[noreturn]] void raise_for(const char* op, const char* msg) {
    raise(PyExc_ValueError, (std::string(op) + ": " + msg).c_str());
}

// The one stride between the rows of [.., n] (0 where there is one row).
int64_t row_stride(const at::Tensor& t, const char* op = "linear") {
    int64_t span = 1, stride = 0;
    for (int64_t d = t.dim() - 2; d >= 0; --d) {
        if (t.size(d) == 1) continue;
        if (t.numel() && span > 1 && t.stride(d) != span * stride)
            raise_for(op, "the rows of a tensor lie at more than one stride");
        if (span == 1) stride = t.stride(d);
        span *= t.size(d);
    }
    return stride;
}

// linear(x, weight, bias | None, out, act, residual | None, stream)
MBRT_PY(linear) {
    HANDLE_TH_ERRORS
    count(n, 7);
    const at::Tensor &x = tensor(a[0]), &w = tensor(a[1]), &out = tensor(a[3]);
    const at::Tensor b = tensor_or_none(a[2]), res = tensor_or_none(a[5]);
    if (x.dim() < 1 || w.dim() != 2 || w.size(1) != x.size(-1))
        raise(PyExc_ValueError, "linear: expected x [.., K] and weight [N, K]");
    const int64_t N = w.size(0), K = w.size(1);
    if (x.scalar_type() != w.scalar_type()) raise(PyExc_ValueError, "linear: x and weight differ in dtype");
    auto fits = [&](const at::Tensor& t) {
        if (t.dim() != x.dim() || t.size(-1) != N) return false;
        for (int64_t d = 0; d < x.dim() - 1; ++d)
            if (t.size(d) != x.size(d)) return false;
        return true;
    };
    if (!fits(out) || (res.defined() && !fits(res))) raise(PyExc_ValueError, "linear: expected out and residual [.., N]");
    if (b.defined() && (b.dim() != 1 || b.size(0) != N)) raise(PyExc_ValueError, "linear: expected bias [N]");
    unit_last({&x, &w, &out, &res, &b});
    int64_t rows = 1;
    for (int64_t d = 0; d < x.dim() - 1; ++d) rows *= x.size(d);
    const int64_t xs = row_stride(x), ws = N > 1 ? w.stride(0) : 0, os = rows > 1 ? row_stride(out) : N;
    const int64_t rs = res.defined() ? row_stride(res) : 0;
    const int dt = dtype_code(x), bd = dtype_or(b, MBRT_F32), rd = dtype_or(res, MBRT_F32), od = dtype_code(out);
    const int act = (int)integer(a[4]);
    void *xp = ptr(x), *wp = ptr(w), *bp = ptr(b), *rp = ptr(res), *op = ptr(out);
    const OnDevice on({&x, &w, &b, &res, &out});
    const mbrt_stream_t st = on.stream(a[6]);
    return call("mbrt_linear",
                [&] { return mbrt_linear(xp, dt, xs, wp, ws, bp, bd, rp, rd, rs, op, od, os, rows, K, N, act, st); });
    END_HANDLE_TH_ERRORS
}

// split_qkv_norm_rotary(qkv, q_gamma, k_gamma, cos, sin, q, k, v | None, heads, kv_heads, scale, eps,
//                       pos0, stream)
MBRT_PY(split_qkv_norm_rotary) {
    HANDLE_TH_ERRORS
    count(n, 14);
    const at::Tensor &qkv = tensor(a[0]), &qg = tensor(a[1]), &kg = tensor(a[2]), &c = tensor(a[3]), &s = tensor(a[4]);
    const at::Tensor &q = tensor(a[5]), &k = tensor(a[6]);
    const at::Tensor v = tensor_or_none(a[7]);
    const int64_t H = integer(a[8]), KV = integer(a[9]);
    if (qkv.dim() != 3 || H < 1 || KV < 1 || qkv.size(2) % (H + 2 * KV))
        raise(PyExc_ValueError, "split_qkv_norm_rotary: expected qkv [B, N, (H + 2 H_kv) D]");
    const int64_t B = qkv.size(0), N = qkv.size(1), D = qkv.size(2) / (H + 2 * KV);
    auto is = [&](const at::Tensor& t, int64_t h) {
        return t.dim() == 4 && t.size(0) == B && t.size(1) == h && t.size(2) == N && t.size(3) == D;
    };
    if (!is(q, H) || !is(k, KV) || (v.defined() && !is(v, KV)))
        raise(PyExc_ValueError, "split_qkv_norm_rotary: expected q [B, H, N, D] and k, v [B, H_kv, N, D]");
    if (q.scalar_type() != k.scalar_type() || (v.defined() && v.scalar_type() != k.scalar_type()))
        raise(PyExc_ValueError, "split_qkv_norm_rotary: q, k and v differ in dtype");
    if (v.defined() && !strided_alike(k, v))
        raise(PyExc_ValueError, "split_qkv_norm_rotary: k and v must be strided alike");
    if (qg.dim() != 1 || qg.size(0) != D || kg.sizes() != qg.sizes() || kg.scalar_type() != qg.scalar_type())
        raise(PyExc_ValueError, "split_qkv_norm_rotary: expected gammas [D] of one dtype");
    if (c.dim() != 2 || c.size(1) != D / 2 || s.sizes() != c.sizes() || s.scalar_type() != c.scalar_type())
        raise(PyExc_ValueError, "split_qkv_norm_rotary: expected cos, sin [n_pos, D/2] of one dtype");
    contig({&qg, &kg, &c, &s});
    unit_last({&qkv, &q, &k, &v});
    const int dt = dtype_code(qkv), gd = dtype_code(qg), td = dtype_code(c), od = dtype_code(q);
    const float scale = (float)number(a[10]), eps = (float)number(a[11]);
    const int64_t pos0 = integer(a[12]), n_pos = c.size(0);
    const int64_t z[8] = {qkv.stride(0), qkv.stride(1), q.stride(0), q.stride(1), q.stride(2),
                          k.stride(0), k.stride(1), k.stride(2)};
    void *xp = ptr(qkv), *qgp = ptr(qg), *kgp = ptr(kg), *cp = ptr(c), *sp = ptr(s), *qp = ptr(q), *kp = ptr(k), *vp = ptr(v);
    const OnDevice on({&qkv, &qg, &kg, &c, &s, &q, &k, &v});
    const mbrt_stream_t st = on.stream(a[13]);
    return call("mbrt_split_qkv_norm_rotary", [&] {
        return mbrt_split_qkv_norm_rotary(xp, dt, z[0], z[1], qgp, kgp, gd, cp, sp, td, n_pos, pos0, qp, kp, vp, od, z[2],
                                          z[3], z[4], z[5], z[6], z[7], B, N, H, KV, D, scale, eps, st);
    });
    END_HANDLE_TH_ERRORS
}

// attention_window(q, k, v, out, left, right, sinks, q_start, key_lens | None, gate | None, gate_is_logit, scale,
//                  workspace | None, stream), -1 for no limit and for queries at the end
MBRT_PY(attention_window) {
    HANDLE_TH_ERRORS
    count(n, 14);
    const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]), &out = tensor(a[3]);
    const at::Tensor lens = tensor_or_none(a[8]), gate = tensor_or_none(a[9]), ws = tensor_or_none(a[12]);
    if (q.dim() != 4 || k.dim() != 4 || k.size(0) != q.size(0) || k.size(3) != q.size(3) || v.sizes() != k.sizes())
        raise(PyExc_ValueError, "attention_window: expected q [B, N_q, H, D] and k, v [B, N_k, H_kv, D]");
    const int64_t B = q.size(0), nq = q.size(1), H = q.size(2), D = q.size(3), nk = k.size(1), KV = k.size(2);
    if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
        raise(PyExc_ValueError, "attention_window: q, k and v differ in dtype");
    if (!strided_alike(k, v)) raise(PyExc_ValueError, "attention_window: k and v must be strided alike");
    if (out.sizes() != q.sizes()) raise(PyExc_ValueError, "attention_window: expected out [B, N_q, H, D]");
    if (lens.defined() && (lens.dim() != 1 || lens.size(0) != B || lens.scalar_type() != at::kInt))
        raise(PyExc_ValueError, "attention_window: expected key_lens [B] int32");
    if (gate.defined() && (gate.dim() != 3 || gate.size(0) != B || gate.size(1) != nq || gate.size(2) != H))
        raise(PyExc_ValueError, "attention_window: expected gate [B, N_q, H]");
    unit_last({&q, &k, &v, &out});
    contig({&lens, &gate, &ws});
    const int dt = dtype_code(q), gd = dtype_or(gate, MBRT_F32), od = dtype_code(out), logit = truth(a[10]);
    const int64_t left = integer(a[4]), right = integer(a[5]), sinks = integer(a[6]), start = integer(a[7]);
    const float scale = (float)number(a[11]);
    const int64_t bytes = ws.defined() ? ws.numel() * (int64_t)ws.element_size() : 0;
    void *qp = ptr(q), *kp = ptr(k), *vp = ptr(v), *op = ptr(out), *gp = ptr(gate), *wp = ptr(ws);
    const int32_t* lp = static_cast<const int32_t*>(ptr(lens));
    const OnDevice on({&q, &k, &v, &out, &lens, &gate, &ws});
    const mbrt_stream_t st = on.stream(a[13]);
    return call("mbrt_attention_window", [&] {
        return mbrt_attention_window(qp, kp, vp, dt, B, H, KV, nq, nk, D, q.stride(0), q.stride(2), q.stride(1),
                                     k.stride(0), k.stride(2), k.stride(1), left, right, sinks, start, lp, gp, gd, logit,
                                     op, od, out.stride(0), out.stride(2), out.stride(1), scale, wp, bytes, st);
    });
    END_HANDLE_TH_ERRORS
}

// Whether t is [*lead of x, n].
bool rows_like(const at::Tensor& t, const at::Tensor& x, int64_t n) {
    if (t.dim() != x.dim() || t.size(-1) != n) return false;
    for (int64_t d = 0; d < x.dim() - 1; ++d)
        if (t.size(d) != x.size(d)) return false;
    return true;
}
int64_t rows_of(const at::Tensor& x) {
    int64_t rows = 1;
    for (int64_t d = 0; d < x.dim() - 1; ++d) rows *= x.size(d);
    return rows;
}

// Row strides of codes and scales that hold rows of n features in 4 bits, as many and shaped as x's.
struct Mx {
    int64_t codes, scales;
};
Mx mx_rows(const char* op, const at::Tensor& codes, const at::Tensor& scales, const at::Tensor& x, int64_t n) {
    if (codes.scalar_type() != at::kByte || scales.scalar_type() != at::kByte)
        raise(PyExc_TypeError, "mbrt: expected codes and scales of dtype torch.uint8");
    const int64_t blocks = (n + 31) / 32;
    if (!rows_like(codes, x, 16 * blocks) || !rows_like(scales, x, blocks))
        raise_for(op, "expected codes [.., 16 ceil(n / 32)] and scales [.., ceil(n / 32)]");
    unit_last({&codes, &scales});
    return Mx{row_stride(codes, op), row_stride(scales, op)};
}

// mx_quantize(x, codes, scales, features, stream)
MBRT_PY(mx_quantize) {
    HANDLE_TH_ERRORS
    count(n, 5);
    const at::Tensor &x = tensor(a[0]), &c = tensor(a[1]), &s = tensor(a[2]);
    const int64_t features = integer(a[3]);
    if (x.dim() < 1 || x.size(-1) != features) raise(PyExc_ValueError, "mx_quantize: expected x [.., n]");
    const Mx m = mx_rows("mx_quantize", c, s, x, features);
    unit_last({&x});
    const int dt = dtype_code(x);
    const int64_t xs = row_stride(x, "mx_quantize"), rows = rows_of(x);
    void *xp = ptr(x), *cp = ptr(c), *sp = ptr(s);
    const OnDevice on({&x, &c, &s});
    const mbrt_stream_t st = on.stream(a[4]);
    return call("mbrt_mx_quantize", [&] { return mbrt_mx_quantize(xp, dt, xs, cp, m.codes, sp, m.scales, rows, features, st); });
    END_HANDLE_TH_ERRORS
}

// mx_dequantize(codes, scales, features, out, stream)
MBRT_PY(mx_dequantize) {
    HANDLE_TH_ERRORS
    count(n, 5);
    const at::Tensor &c = tensor(a[0]), &s = tensor(a[1]), &out = tensor(a[3]);
    const int64_t features = integer(a[2]);
    if (out.dim() < 1 || out.size(-1) != features) raise(PyExc_ValueError, "mx_dequantize: expected out [.., n]");
    const Mx m = mx_rows("mx_dequantize", c, s, out, features);
    unit_last({&out});
    const int dt = dtype_code(out);
    const int64_t os = row_stride(out, "mx_dequantize"), rows = rows_of(out);
    void *cp = ptr(c), *sp = ptr(s), *op = ptr(out);
    const OnDevice on({&c, &s, &out});
    const mbrt_stream_t st = on.stream(a[4]);
    return call("mbrt_mx_dequantize",
                [&] { return mbrt_mx_dequantize(cp, m.codes, sp, m.scales, op, dt, os, rows, features, st); });
    END_HANDLE_TH_ERRORS
}

// mx_linear(x, x_scales | None, weight codes, weight scales, K, bias | None, out, out_scales | None, act, residual | None,
//           stream), with scales where x or out is in 4 bits
MBRT_PY(mx_linear) {
    HANDLE_TH_ERRORS
    count(n, 11);
    const char* name = "mx_linear";
    const at::Tensor &x = tensor(a[0]), &w = tensor(a[2]), &wsc = tensor(a[3]), &out = tensor(a[6]);
    const at::Tensor xsc = tensor_or_none(a[1]), b = tensor_or_none(a[5]), osc = tensor_or_none(a[7]), res = tensor_or_none(a[9]);
    const int64_t K = integer(a[4]);
    if (x.dim() < 1 || w.dim() != 2 || (!xsc.defined() && x.size(-1) != K))
        raise(PyExc_ValueError, "mx_linear: expected x [.., K] and weight [N, K]");
    const int64_t N = w.size(0), rows = rows_of(x);
    const Mx wm = mx_rows(name, w, wsc, w, K);
    const Mx xm = xsc.defined() ? mx_rows(name, x, xsc, x, K) : Mx{row_stride(x, name), 0};
    if ((!osc.defined() && !rows_like(out, x, N)) || (res.defined() && !rows_like(res, x, N)))
        raise(PyExc_ValueError, "mx_linear: expected out and residual [.., N]");
    const Mx om = osc.defined() ? mx_rows(name, out, osc, x, N) : Mx{row_stride(out, name), 0};
    if (b.defined() && (b.dim() != 1 || b.size(0) != N)) raise(PyExc_ValueError, "mx_linear: expected bias [N]");
    unit_last({&x, &out, &res, &b});
    const int xd = xsc.defined() ? MBRT_MXFP4 : dtype_code(x), od = osc.defined() ? MBRT_MXFP4 : dtype_code(out);
    const int bd = dtype_or(b, MBRT_F32), rd = dtype_or(res, MBRT_F32), act = (int)integer(a[8]);
    const int64_t rs = res.defined() ? row_stride(res, name) : 0;
    void *xp = ptr(x), *xsp = ptr(xsc), *wp = ptr(w), *wsp = ptr(wsc), *bp = ptr(b), *rp = ptr(res), *op = ptr(out), *osp = ptr(osc);
    const OnDevice on({&x, &xsc, &w, &wsc, &b, &res, &out, &osc});
    const mbrt_stream_t st = on.stream(a[10]);
    return call("mbrt_mx_linear", [&] {
        return mbrt_mx_linear(xp, xd, xm.codes, xsp, xm.scales, wp, wm.codes, wsp, wm.scales, bp, bd, rp, rd, rs, op, od, om.codes,
                              osp, om.scales, rows, K, N, act, st);
    });
    END_HANDLE_TH_ERRORS
}

// Row r of `like` [.., D] has the gate's row (r / inner) % period.
struct GateRows {
    int64_t cols = 1, stride = 0, inner = 1, period = 1;
};
GateRows gate_rows(const at::Tensor& gate, const at::Tensor& like) {
    GateRows r;
    if (!gate.defined()) return r;
    const char* shape = "expected gate [.., D] or [.., 1]";
    if (gate.dim() < 1 || gate.dim() > like.dim() || (gate.size(-1) != 1 && gate.size(-1) != like.size(-1)))
        raise_for("block_norm", shape);
    r.cols = gate.size(-1);
    bool closed = false;
    for (int64_t d = 2; d <= like.dim(); ++d) {
        const int64_t n = like.size(-d), m = d <= gate.dim() ? gate.size(-d) : 1;
        if (m != 1 && m != n) raise_for("block_norm", shape);
        if (n == 1) continue;
        if (m == 1) {
            if (r.period == 1) r.inner *= n;
            else closed = true;
            continue;
        }
        if (closed) raise_for("block_norm", "the gate's rows are shared on both sides of a dim that they do not share");
        if (r.period > 1 && like.numel() && gate.stride(-d) != r.period * r.stride)
            raise_for("block_norm", "the rows of a tensor lie at more than one stride");
        if (r.period == 1) r.stride = gate.stride(-d);
        r.period *= n;
    }
    if (r.inner < 1) r.inner = 1;
    if (r.period < 1) r.period = 1;
    return r;
}

// block_norm(residual, update, post_gamma | None, gate | None, gate_is_logit, layer_scale | None, gamma | None, sum_out | None,
//            normed | None, normed_scales | None, alpha, post_scale, scale, eps, stream)
MBRT_PY(block_norm) {
    HANDLE_TH_ERRORS
    count(n, 15);
    const char* name = "block_norm";
    const at::Tensor &res = tensor(a[0]), &upd = tensor(a[1]);
    const at::Tensor pg = tensor_or_none(a[2]), gate = tensor_or_none(a[3]), ls = tensor_or_none(a[5]), g = tensor_or_none(a[6]);
    const at::Tensor sum = tensor_or_none(a[7]), out = tensor_or_none(a[8]), osc = tensor_or_none(a[9]);
    auto fits = [&](const at::Tensor& t) { return !t.defined() || t.sizes() == res.sizes(); };
    if (res.dim() < 1 || res.size(-1) < 1 || !fits(upd) || !fits(sum) || (!osc.defined() && !fits(out)))
        raise(PyExc_ValueError, "block_norm: expected update, sum_out and normed [.., D]");
    if (sum.defined() && sum.scalar_type() != res.scalar_type())
        raise(PyExc_ValueError, "block_norm: sum_out and residual differ in dtype");
    const int64_t D = res.size(-1), rows = rows_of(res);
    for (const at::Tensor* t : {&pg, &ls, &g})
        if (t->defined() && (t->dim() != 1 || t->size(0) != D))
            raise(PyExc_ValueError, "block_norm: expected gammas and layer_scale [D]");
    contig({&pg, &ls, &g});
    unit_last({&res, &upd, &sum, &out, &gate});
    const Mx om = !out.defined() ? Mx{0, 0} : osc.defined() ? mx_rows(name, out, osc, res, D) : Mx{row_stride(out, name), 0};
    const int od = osc.defined() ? MBRT_MXFP4 : dtype_or(out, MBRT_F32);
    const GateRows gr = gate_rows(gate, res);
    const int rd = dtype_code(res), ud = dtype_code(upd), pd = dtype_or(pg, MBRT_F32), gd = dtype_or(gate, MBRT_F32);
    const int ld = dtype_or(ls, MBRT_F32), gad = dtype_or(g, MBRT_F32), logit = truth(a[4]);
    const int64_t rs = row_stride(res, name), us = row_stride(upd, name), ss = sum.defined() ? row_stride(sum, name) : 0;
    const float alpha = (float)number(a[10]), ps = (float)number(a[11]), sc = (float)number(a[12]), eps = (float)number(a[13]);
    void *rp = ptr(res), *up = ptr(upd), *pp = ptr(pg), *gp = ptr(gate), *lp = ptr(ls), *gap = ptr(g), *sp = ptr(sum),
         *op = ptr(out), *osp = ptr(osc);
    const OnDevice on({&res, &upd, &pg, &gate, &ls, &g, &sum, &out, &osc});
    const mbrt_stream_t st = on.stream(a[14]);
    return call("mbrt_block_norm", [&] {
        return mbrt_block_norm(rp, rd, rs, up, ud, us, pp, pd, gp, gd, gr.cols, gr.stride, gr.inner, gr.period, logit, lp, ld,
                               gap, gad, sp, ss, op, od, om.codes, osp, om.scales, rows, D, alpha, ps, sc, eps, st);
    });
    END_HANDLE_TH_ERRORS
}

// stft(x [B, L], window, hop, center, normalized, out, n_fft, win_length, stream)
MBRT_PY(stft) {
    HANDLE_TH_ERRORS
    count(n, 9);
    const at::Tensor &x = tensor(a[0]), &w = tensor(a[1]), &out = tensor(a[5]);
    contig({&x, &w, &out});
    const int64_t hop = integer(a[2]), n_fft = integer(a[6]), win = integer(a[7]);
    const int center = truth(a[3]), normalized = truth(a[4]);
    const int64_t B = x.size(0), L = x.size(1), wn = w.numel();
    const float *xp = static_cast<const float*>(ptr(x)), *wp = static_cast<const float*>(ptr(w));
    float* op = static_cast<float*>(ptr(out));
    const mbrt_stream_t st = stream(a[8]);
    return call("mbrt_stft", [&] { return mbrt_stft(xp, wp, op, B, L, n_fft, hop, win, wn, center, normalized, st); });
    END_HANDLE_TH_ERRORS
}

// istft(spec, window, hop, center, normalized, length, out, workspace, n_fft, win_length, stream)
MBRT_PY(istft) {
    HANDLE_TH_ERRORS
    count(n, 11);
    const at::Tensor &s = tensor(a[0]), &w = tensor(a[1]), &out = tensor(a[6]), &ws = tensor(a[7]);
    contig({&s, &w, &out});
    if (s.dim() != 4) raise(PyExc_ValueError, "istft: expected a spectrum [B, F, T, 2]");
    const int64_t hop = integer(a[2]), length = integer(a[5]), n_fft = integer(a[8]), win = integer(a[9]);
    const int center = truth(a[3]), normalized = truth(a[4]), dt = dtype_code(s);
    const int64_t B = s.size(0), F = s.size(1), T = s.size(2), wn = w.numel();
    const int64_t bytes = ws.numel() * (int64_t)ws.element_size();
    void *sp = ptr(s), *wsp = ptr(ws);
    const float* wp = static_cast<const float*>(ptr(w));
    float* op = static_cast<float*>(ptr(out));
    const mbrt_stream_t st = stream(a[10]);
    return call("mbrt_istft", [&] {
        return mbrt_istft(sp, dt, wp, op, B, F, T, n_fft, hop, win, wn, center, normalized, length, wsp, bytes, st);
    });
    END_HANDLE_TH_ERRORS
}

// chunk_accumulate(dest, weight_sum, src, window, offset, stream)
MBRT_PY(chunk_accumulate) {
    HANDLE_TH_ERRORS
    count(n, 6);
    const at::Tensor &d = tensor(a[0]), &ws = tensor(a[1]), &s = tensor(a[2]), &w = tensor(a[3]);
    contig({&d, &ws, &s, &w});
    const int64_t len = s.size(-1), L = d.size(-1), off = integer(a[4]);
    const int64_t channels = s.numel() / (len > 1 ? len : 1);
    float *dp = static_cast<float*>(ptr(d)), *wsp = static_cast<float*>(ptr(ws));
    const float *sp = static_cast<const float*>(ptr(s)), *wp = static_cast<const float*>(ptr(w));
    const mbrt_stream_t st = stream(a[5]);
    return call("mbrt_chunk_accumulate",
                [&] { return mbrt_chunk_accumulate(dp, wsp, sp, wp, channels, len, L, off, st); });
    END_HANDLE_TH_ERRORS
}

// init(MbrtError)
MBRT_PY(init) {
    HANDLE_TH_ERRORS
    count(n, 1);
    Py_INCREF(a[0]);
    Py_XDECREF(g_error);
    g_error = a[0];
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

#define MBRT_DEF(fname) {#fname, (PyCFunction)(void (*)(void))fname, METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {
    MBRT_DEF(init), MBRT_DEF(fill), MBRT_DEF(strided_copy), MBRT_DEF(pad), MBRT_DEF(cat), MBRT_DEF(rms_norm),
    MBRT_DEF(residual_add_rms_norm), MBRT_DEF(bias_act), MBRT_DEF(glu), MBRT_DEF(gate_merge), MBRT_DEF(softmax),
    MBRT_DEF(split_qkv_rotary), MBRT_DEF(attention_ex), MBRT_DEF(stft), MBRT_DEF(istft), MBRT_DEF(chunk_accumulate),
    MBRT_DEF(linear), MBRT_DEF(split_qkv_norm_rotary), MBRT_DEF(attention_window),
    MBRT_DEF(mx_quantize), MBRT_DEF(mx_dequantize), MBRT_DEF(mx_linear), MBRT_DEF(block_norm),
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_mbrt_calls", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__mbrt_calls(void) { return PyModule_Create(&kModule); }
