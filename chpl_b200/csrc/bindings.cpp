// Python bindings of the entry points of a model's layers for torch tensors: the
// module chpl_b200._torch, which chpl_b200/ckpt8.py, linear.py, norm.py and mx4.py
// call.
//
// A one-token product takes the GPU about as long as a ctypes call takes the
// host, so here the tensors' shapes, strides and devices are read, and the
// outputs allocated, in C++ (a forward call: 9 us of host time by ctypes, 5 by
// this; the launch itself is 3).  Every function takes its arguments by position;
// None stands for what is not given.  All work is queued on torch's current
// stream of the tensors' device, whose memory outputs and workspaces come from.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>

#include "chpl.h"

namespace {

constexpr int64_t kGroup = 32;

// chpl_b200._lib.ChplError(code, where, message) as the pending Python error
struct Raised {};

[[noreturn]] void raise(int code, const char* where, const char* fmt, ...)
{
    char msg[512];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(msg, sizeof(msg), fmt, ap);
    va_end(ap);
    PyObject* lib = PyImport_ImportModule("chpl_b200._lib");
    PyObject* cls = lib ? PyObject_GetAttrString(lib, "ChplError") : nullptr;
    PyObject* err = cls ? PyObject_CallFunction(cls, "iss", code, where, msg) : nullptr;
    if (err) PyErr_SetObject(cls, err);
    Py_XDECREF(err);
    Py_XDECREF(cls);
    Py_XDECREF(lib);
    throw Raised();
}

void check(int code, const char* where)
{
    if (code != CHPL_OK) raise(code, where, "%s", chpl_last_error_string());
}

// Guards a function called from Python: C++ exceptions become Python's.
#define CHPL_PY_BEGIN HANDLE_TH_ERRORS try {
#define CHPL_PY_END                      \
    }                                    \
    catch (const Raised&) { return nullptr; } \
    END_HANDLE_TH_ERRORS

bool given(PyObject* o) { return o != Py_None; }

int type_code(at::ScalarType t)
{
    return t == at::kBFloat16 ? CHPL_TYPE_BF16 : t == at::kHalf ? CHPL_TYPE_F16 : t == at::kFloat ? CHPL_TYPE_F32 : -1;
}

const at::Tensor& tensor(const char* where, const char* name, PyObject* o, int dim)
{
    if (!THPVariable_Check(o)) raise(CHPL_ERR_INVALID, where, "%s is not a tensor", name);
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.dim() != dim) raise(CHPL_ERR_INVALID, where, "%s is not a %s", name, dim == 2 ? "matrix" : "vector");
    if (!t.is_cuda()) raise(CHPL_ERR_INVALID, where, "%s is not on a GPU", name);
    return t;
}

// distance between the rows of a matrix whose rows are contiguous
int64_t row_distance(const char* where, const char* name, const at::Tensor& t)
{
    const int64_t rows = t.size(0), cols = t.size(1);
    if (cols > 1 && t.stride(1) != 1) raise(CHPL_ERR_INVALID, where, "%s has column stride %lld: rows must be contiguous", name, (long long)t.stride(1));
    if (rows > 1 && t.stride(0) < cols) raise(CHPL_ERR_INVALID, where, "%s has row stride %lld below its %lld columns", name, (long long)t.stride(0), (long long)cols);
    return rows > 1 ? t.stride(0) : cols;
}

// What sets a call's type and device, and checks the other tensors against it.
struct Call {
    const char* where;
    at::ScalarType type;
    at::Device device;
    c10::cuda::OptionalCUDAGuard guard;  // set where the tensors' device is not the current one

    Call(const char* who, const at::Tensor& t) : where(who), type(t.scalar_type()), device(t.device())
    {
        if (device.index() != c10::cuda::current_device()) guard.set_device(device);
    }
    void* stream() const { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }
    // (past the dispatcher, which costs more than the allocation; a TorchDispatchMode does not see these, and
    // torch.utils.deterministic.fill_uninitialized_memory does not fill them: every element is written by the call)
    at::Tensor empty(int64_t rows, int64_t cols, at::ScalarType t) const { return at::detail::empty_cuda({rows, cols}, t, device, c10::nullopt); }
    at::Tensor empty(int64_t n, at::ScalarType t) const { return at::detail::empty_cuda({n}, t, device, c10::nullopt); }

    void same(const char* name, const at::Tensor& t, at::ScalarType type) const
    {
        if (t.scalar_type() != type) raise(CHPL_ERR_INVALID, where, "%s is %s, not %s", name, at::toString(t.scalar_type()), at::toString(type));
        if (t.device() != device) raise(CHPL_ERR_INVALID, where, "%s is on another device", name);
    }
    const at::Tensor& matrix(const char* name, PyObject* o, at::ScalarType type, int64_t rows, int64_t cols, int64_t* ld) const
    {
        const at::Tensor& t = tensor(where, name, o, 2);
        same(name, t, type);
        if (t.size(0) != rows || t.size(1) != cols)
            raise(CHPL_ERR_INVALID, where, "%s is %lld x %lld, not %lld x %lld", name, (long long)t.size(0), (long long)t.size(1), (long long)rows, (long long)cols);
        *ld = row_distance(where, name, t);
        return t;
    }
    const at::Tensor& vector(const char* name, PyObject* o, at::ScalarType type, int64_t n) const
    {
        const at::Tensor& t = tensor(where, name, o, 1);
        same(name, t, type);
        if (t.size(0) != n || (n > 1 && t.stride(0) != 1)) raise(CHPL_ERR_INVALID, where, "%s is not a contiguous vector of %lld", name, (long long)n);
        return t;
    }
    chpl_ckpt8 checkpoint(const char* name, PyObject* codes, PyObject* scales, int64_t rows, int64_t cols) const
    {
        chpl_ckpt8 c;
        char part[64];
        std::snprintf(part, sizeof(part), "%s.codes", name);
        c.codes = static_cast<int8_t*>(matrix(part, codes, at::kChar, rows, cols, &c.ldc).data_ptr());
        std::snprintf(part, sizeof(part), "%s.scales", name);
        c.scales = static_cast<uint8_t*>(matrix(part, scales, at::kByte, rows, (cols + kGroup - 1) / kGroup, &c.lds).data_ptr());
        return c;
    }
};

// a new checkpoint's tensors; rows of codes a multiple of 16 bytes apart, which
// the kernels read and write in whole pieces
struct NewCkpt {
    at::Tensor codes, scales;
    chpl_ckpt8 make(const Call& call, int64_t rows, int64_t cols)
    {
        const int64_t groups = (cols + kGroup - 1) / kGroup, ld = (cols + 15) / 16 * 16;
        codes = call.empty(rows, ld, at::kChar);
        if (ld != cols) codes = codes.as_strided({rows, cols}, {ld, 1});
        scales = call.empty(rows, groups, at::kByte);
        return {static_cast<int8_t*>(codes.data_ptr()), static_cast<uint8_t*>(scales.data_ptr()), ld, groups};
    }
};

PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }
PyObject* same_object(PyObject* o)
{
    Py_INCREF(o);
    return o;
}

void arguments(const char* where, Py_ssize_t n, Py_ssize_t want)
{
    if (n != want) raise(CHPL_ERR_INVALID, where, "%lld arguments, %lld are wanted", (long long)n, (long long)want);
}

// memory that chpl_linear_* works in: the caller's, or new
struct Workspace {
    at::Tensor own;
    void* at = nullptr;
    size_t bytes = 0;
    Workspace(const Call& call, PyObject* work, size_t need)
    {
        if (given(work)) {
            if (!THPVariable_Check(work)) raise(CHPL_ERR_INVALID, call.where, "work is not a tensor");
            const at::Tensor& t = THPVariable_Unpack(work);
            if (t.device() != call.device || !t.is_contiguous()) raise(CHPL_ERR_INVALID, call.where, "work is not contiguous memory of the tensors' device");
            at = t.data_ptr();
            bytes = t.nbytes();
        } else if (need) {
            own = call.empty((int64_t)need, at::kByte);
            at = own.data_ptr();
            bytes = need;
        }
    }
};

// ckpt8_pack(x, codes, scales) -> (codes, scales)
PyObject* ckpt8_pack(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    CHPL_PY_BEGIN
    const char* where = "ckpt8.pack";
    arguments(where, n, 3);
    const at::Tensor& x = tensor(where, "x", a[0], 2);
    const int type = type_code(x.scalar_type());
    if (type < 0) raise(CHPL_ERR_INVALID, where, "x is %s: bfloat16, float16 or float32 is wanted", at::toString(x.scalar_type()));
    const int64_t ldx = row_distance(where, "x", x), rows = x.size(0), cols = x.size(1);
    const Call call(where, x);
    NewCkpt made;
    const chpl_ckpt8 c = given(a[1]) ? call.checkpoint("out", a[1], a[2], rows, cols) : made.make(call, rows, cols);
    check(chpl_ckpt8_pack(call.stream(), type, rows, cols, x.data_ptr(), ldx, &c), "chpl_ckpt8_pack");
    if (given(a[1])) return PyTuple_Pack(2, a[1], a[2]);
    return Py_BuildValue("NN", wrap(std::move(made.codes)), wrap(std::move(made.scales)));
    CHPL_PY_END
}

// ckpt8_unpack(codes, scales, dtype, out) -> x
PyObject* ckpt8_unpack(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    CHPL_PY_BEGIN
    const char* where = "ckpt8.unpack";
    arguments(where, n, 4);
    const at::Tensor& codes = tensor(where, "c.codes", a[0], 2);
    const int64_t rows = codes.size(0), cols = codes.size(1);
    const Call call(where, codes);
    const chpl_ckpt8 c = call.checkpoint("c", a[0], a[1], rows, cols);
    if (!THPDtype_Check(a[2])) raise(CHPL_ERR_INVALID, where, "dtype is not a torch.dtype");
    const at::ScalarType to = reinterpret_cast<THPDtype*>(a[2])->scalar_type;
    const int type = type_code(to);
    if (type < 0) raise(CHPL_ERR_INVALID, where, "%s: bfloat16, float16 or float32 is wanted", at::toString(to));
    int64_t ldx = cols;
    at::Tensor x = given(a[3]) ? call.matrix("out", a[3], to, rows, cols, &ldx) : call.empty(rows, cols, to);
    check(chpl_ckpt8_unpack(call.stream(), type, rows, cols, &c, x.data_ptr(), ldx), "chpl_ckpt8_unpack");
    return given(a[3]) ? same_object(a[3]) : wrap(std::move(x));
    CHPL_PY_END
}

// linear_forward(x, w, bias, residual, act, save, out, z, z.codes, z.scales, work)
//   -> Y; with save 1 (Y, Z), with save 2 (Y, codes, scales)
PyObject* linear_forward(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    CHPL_PY_BEGIN
    const char* where = "linear.forward";
    arguments(where, n, 11);
    const at::Tensor &x = tensor(where, "x", a[0], 2), &w = tensor(where, "w", a[1], 2);
    chpl_linear_fwd f = {};
    f.type = type_code(x.scalar_type());
    f.act = (int)PyLong_AsLong(a[4]);
    const long save = PyLong_AsLong(a[5]);
    if (PyErr_Occurred()) return nullptr;
    f.tokens = x.size(0);
    f.k = x.size(1);
    f.n = w.size(0);
    const Call call(where, x);
    if (w.size(1) != f.k) raise(CHPL_ERR_INVALID, where, "x has %lld features and w %lld", (long long)f.k, (long long)w.size(1));
    call.same("w", w, call.type);
    f.x = x.data_ptr();
    f.ldx = row_distance(where, "x", x);
    f.w = w.data_ptr();
    f.ldw = row_distance(where, "w", w);
    if (given(a[2])) f.bias = call.vector("bias", a[2], call.type, f.n).data_ptr();
    if (given(a[3])) f.residual = call.matrix("residual", a[3], call.type, f.tokens, f.n, &f.ldr).data_ptr();
    f.ldy = f.ldz = f.n;
    at::Tensor y = given(a[6]) ? call.matrix("out", a[6], call.type, f.tokens, f.n, &f.ldy) : call.empty(f.tokens, f.n, call.type);
    f.y = y.data_ptr();
    at::Tensor z;
    NewCkpt z8;
    if (save == 1) {
        z = given(a[7]) ? call.matrix("z", a[7], call.type, f.tokens, f.n, &f.ldz) : call.empty(f.tokens, f.n, call.type);
        f.z = z.data_ptr();
    } else if (save == 2) {
        f.z8 = given(a[8]) ? call.checkpoint("z", a[8], a[9], f.tokens, f.n) : z8.make(call, f.tokens, f.n);
    }
    size_t need = 0;
    check(chpl_linear_forward_worksize(&f, &need), "chpl_linear_forward_worksize");
    const Workspace work(call, a[10], need);
    check(chpl_linear_forward(call.stream(), &f, work.at, work.bytes), "chpl_linear_forward");
    PyObject* out = given(a[6]) ? same_object(a[6]) : wrap(std::move(y));
    if (save == 1) return Py_BuildValue("NN", out, given(a[7]) ? same_object(a[7]) : wrap(std::move(z)));
    if (save == 2) {
        if (given(a[8])) return Py_BuildValue("NOO", out, a[8], a[9]);
        return Py_BuildValue("NNN", out, wrap(std::move(z8.codes)), wrap(std::move(z8.scales)));
    }
    return out;
    CHPL_PY_END
}

// linear_backward(dy, w, x, x.codes, x.scales, z, z.codes, z.scales, add, act, in_act, float32 gradients, accumulate,
//                 need dx, need dw, need db, need dx_sum, dx, dw, db, dx_sum, work) -> (dx, dw, db, dx_sum)
PyObject* linear_backward(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    CHPL_PY_BEGIN
    const char* where = "linear.backward";
    arguments(where, n, 22);
    const at::Tensor &dy = tensor(where, "dy", a[0], 2), &w = tensor(where, "w", a[1], 2);
    chpl_linear_bwd b = {};
    b.type = type_code(dy.scalar_type());
    b.act = (int)PyLong_AsLong(a[9]);
    b.in_act = (int)PyLong_AsLong(a[10]);
    if (PyErr_Occurred()) return nullptr;
    const bool f32 = PyObject_IsTrue(a[11]), dx_wanted = PyObject_IsTrue(a[13]), dw_wanted = PyObject_IsTrue(a[14]),
               db_wanted = PyObject_IsTrue(a[15]), sum_wanted = PyObject_IsTrue(a[16]);
    b.accumulate = PyObject_IsTrue(a[12]);
    b.grad_type = f32 ? CHPL_TYPE_F32 : b.type;
    const at::ScalarType gt = f32 ? at::kFloat : dy.scalar_type();
    b.tokens = dy.size(0);
    b.n = dy.size(1);
    b.k = w.size(1);
    const Call call(where, dy);
    if (w.size(0) != b.n) raise(CHPL_ERR_INVALID, where, "dy has %lld features and w %lld rows", (long long)b.n, (long long)w.size(0));
    call.same("w", w, call.type);
    b.dy = dy.data_ptr();
    b.lddy = row_distance(where, "dy", dy);
    b.w = w.data_ptr();
    b.ldw = row_distance(where, "w", w);
    if (given(a[2])) b.x = call.matrix("x", a[2], call.type, b.tokens, b.k, &b.ldx).data_ptr();
    if (given(a[3])) b.x8 = call.checkpoint("x", a[3], a[4], b.tokens, b.k);
    if (b.act != CHPL_ACT_NONE) {
        if (given(a[5])) b.z = call.matrix("z", a[5], call.type, b.tokens, b.n, &b.ldz).data_ptr();
        if (given(a[6])) b.z8 = call.checkpoint("z", a[6], a[7], b.tokens, b.n);
    }
    if (given(a[8])) b.add = call.matrix("add", a[8], call.type, b.tokens, b.k, &b.ldadd).data_ptr();
    b.lddx = b.lddw = b.k;
    at::Tensor dx, dw, db, sum;
    if (dx_wanted) {
        dx = given(a[17]) ? call.matrix("dx", a[17], call.type, b.tokens, b.k, &b.lddx) : call.empty(b.tokens, b.k, call.type);
        b.dx = dx.data_ptr();
    }
    if (dw_wanted) {
        dw = given(a[18]) ? call.matrix("dw", a[18], gt, b.n, b.k, &b.lddw) : call.empty(b.n, b.k, gt);
        b.dw = dw.data_ptr();
    }
    if (db_wanted) {
        db = given(a[19]) ? call.vector("db", a[19], gt, b.n) : call.empty(b.n, gt);
        b.db = db.data_ptr();
    }
    if (sum_wanted) {
        sum = given(a[20]) ? call.vector("dx_sum", a[20], gt, b.k) : call.empty(b.k, gt);
        b.dx_sum = sum.data_ptr();
    }
    size_t need = 0;
    check(chpl_linear_backward_worksize(&b, &need), "chpl_linear_backward_worksize");
    const Workspace work(call, a[21], need);
    check(chpl_linear_backward(call.stream(), &b, work.at, work.bytes), "chpl_linear_backward");
    const auto result = [&](bool wanted, PyObject* mine, at::Tensor& t) {
        return !wanted ? same_object(Py_None) : given(mine) ? same_object(mine) : wrap(std::move(t));
    };
    PyObject *px = result(dx_wanted, a[17], dx), *pw = result(dw_wanted, a[18], dw), *pb = result(db_wanted, a[19], db),
             *ps = result(sum_wanted, a[20], sum);
    return Py_BuildValue("NNNN", px, pw, pb, ps);
    CHPL_PY_END
}

// ----------------------------------------------------------------------------
// norms
// ----------------------------------------------------------------------------
double number(PyObject* o)
{
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}

// kind, weight, bias, eps of a norm; kind 0: none
chpl_norm norm_of(const Call& call, const char* name, PyObject* const* a, int64_t n)
{
    chpl_norm v = {};
    v.kind = (int)number(a[0]);
    if (v.kind == CHPL_NORM_NONE) return v;
    char part[64];
    std::snprintf(part, sizeof(part), "%s.weight", name);
    v.weight = call.vector(part, a[1], call.type, n).data_ptr();
    std::snprintf(part, sizeof(part), "%s.bias", name);
    if (given(a[2])) v.bias = call.vector(part, a[2], call.type, n).data_ptr();
    v.eps = (float)number(a[3]);
    return v;
}

float* statistics(const Call& call, const char* name, PyObject* o, int64_t tokens)
{
    int64_t ld = 0;
    const at::Tensor& t = call.matrix(name, o, at::kFloat, tokens, 2, &ld);
    if (!t.is_contiguous()) raise(CHPL_ERR_INVALID, call.where, "%s is not contiguous", name);
    return static_cast<float*>(t.data_ptr());
}

// a gate: a vector, or a row for each token; ld 0: a vector
const void* gate_of(const Call& call, PyObject* o, int64_t tokens, int64_t n, int64_t* ld)
{
    *ld = 0;
    if (!given(o)) return nullptr;
    if (!THPVariable_Check(o)) raise(CHPL_ERR_INVALID, call.where, "gate is not a tensor");
    if (THPVariable_Unpack(o).dim() == 1) {
        if (!THPVariable_Unpack(o).is_cuda()) raise(CHPL_ERR_INVALID, call.where, "gate is not on a GPU");
        return call.vector("gate", o, call.type, n).data_ptr();
    }
    const void* p = call.matrix("gate", o, call.type, tokens, n, ld).data_ptr();
    *ld = std::max<int64_t>(*ld, 1);
    return p;
}

// norm_forward(join, x, y, gate, scale, residual_scale, post: kind, weight, bias, eps, pre: kind, weight, bias, eps, save, r, h)
//   -> (r, h, post statistics, pre statistics)
PyObject* norm_forward(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    CHPL_PY_BEGIN
    const bool join = n > 0 && PyObject_IsTrue(a[0]);
    const char* where = join ? "norm.join" : "norm.forward";
    arguments(where, n, 17);
    const at::Tensor& x = tensor(where, "x", a[1], 2);
    chpl_norm_fwd f = {};
    f.type = type_code(x.scalar_type());
    f.join = join;
    f.tokens = x.size(0);
    f.n = x.size(1);
    const Call call(where, x);
    f.x = x.data_ptr();
    f.ldx = row_distance(where, "x", x);
    f.pre = norm_of(call, join ? "pre" : "norm", a + 10, f.n);
    const bool save = PyObject_IsTrue(a[14]);
    at::Tensor r, h, post_stats, pre_stats;
    if (join) {
        f.y = call.matrix("y", a[2], call.type, f.tokens, f.n, &f.ldy).data_ptr();
        f.gate = gate_of(call, a[3], f.tokens, f.n, &f.ldgate);
        f.scale = (float)number(a[4]);
        f.residual_scale = (float)number(a[5]);
        f.post = norm_of(call, "post", a + 6, f.n);
        f.ldr = f.n;
        r = given(a[15]) ? call.matrix("out", a[15], call.type, f.tokens, f.n, &f.ldr) : call.empty(f.tokens, f.n, call.type);
        f.r = r.data_ptr();
        if (save && f.post.kind) {
            post_stats = call.empty(f.tokens, 2, at::kFloat);
            f.post_stats = static_cast<float*>(post_stats.data_ptr());
        }
    }
    if (f.pre.kind) {
        f.ldh = f.n;
        h = given(a[16]) ? call.matrix("out", a[16], call.type, f.tokens, f.n, &f.ldh) : call.empty(f.tokens, f.n, call.type);
        f.h = h.data_ptr();
        if (save) {
            pre_stats = call.empty(f.tokens, 2, at::kFloat);
            f.pre_stats = static_cast<float*>(pre_stats.data_ptr());
        }
    }
    check(chpl_norm_forward(call.stream(), &f), "chpl_norm_forward");
    const auto result = [](PyObject* mine, at::Tensor& t) { return !t.defined() ? same_object(Py_None) : given(mine) ? same_object(mine) : wrap(std::move(t)); };
    PyObject *pr = result(a[15], r), *ph = result(a[16], h), *ps = result(Py_None, post_stats), *pp = result(Py_None, pre_stats);
    return Py_BuildValue("NNNN", pr, ph, ps, pp);
    CHPL_PY_END
}

// norm_backward(join, dr, dh, r, y, gate, scale, residual_scale, post: kind, weight, bias, eps, pre: kind, weight, bias, eps,
//               post statistics, pre statistics, float32 gradients, accumulate, need dx, dy, dgate, parameters,
//               dx, dy, dgate, post dweight, post dbias, pre dweight, pre dbias, work)
//   -> (dx, dy, dgate, post dweight, post dbias, pre dweight, pre dbias)
PyObject* norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    CHPL_PY_BEGIN
    const bool join = n > 0 && PyObject_IsTrue(a[0]);
    const char* where = join ? "norm.join_backward" : "norm.backward";
    arguments(where, n, 32);
    if (!given(a[1]) && !given(a[2])) raise(CHPL_ERR_INVALID, where, "neither dr nor dh");
    const at::Tensor& d = given(a[2]) ? tensor(where, "dh", a[2], 2) : tensor(where, "dr", a[1], 2);
    chpl_norm_bwd b = {};
    b.type = type_code(d.scalar_type());
    b.join = join;
    b.tokens = d.size(0);
    b.n = d.size(1);
    const Call call(where, d);
    if (given(a[1])) b.dr = call.matrix(join ? "dr" : "add", a[1], call.type, b.tokens, b.n, &b.lddr).data_ptr();
    b.pre = norm_of(call, join ? "pre" : "norm", a + 12, b.n);
    if ((b.pre.kind != 0) != given(a[2])) raise(CHPL_ERR_INVALID, where, b.pre.kind ? "dh is missing" : "dh without a norm of the sum");
    if (b.pre.kind) {
        b.dh = call.matrix("dh", a[2], call.type, b.tokens, b.n, &b.lddh).data_ptr();
        b.r = call.matrix(join ? "r" : "x", a[3], call.type, b.tokens, b.n, &b.ldr).data_ptr();
        b.pre_stats = statistics(call, join ? "pre_stats" : "stats", a[17], b.tokens);
    }
    b.scale = (float)number(a[6]);
    b.residual_scale = (float)number(a[7]);
    const bool f32 = PyObject_IsTrue(a[18]);
    b.accumulate = PyObject_IsTrue(a[19]);
    b.grad_type = f32 ? CHPL_TYPE_F32 : b.type;
    const at::ScalarType gt = f32 ? at::kFloat : call.type;
    const bool params = PyObject_IsTrue(a[23]);
    at::Tensor dx, dy, dgate, sums[4];
    const auto rows_to = [&](const char* name, bool wanted, PyObject* mine, at::Tensor& t, void*& p, int64_t& ld) {
        if (!wanted) return;
        ld = b.n;
        t = given(mine) ? call.matrix(name, mine, call.type, b.tokens, b.n, &ld) : call.empty(b.tokens, b.n, call.type);
        p = t.data_ptr();
    };
    const auto sum_to = [&](const char* name, bool wanted, PyObject* mine, at::Tensor& t, void*& p) {
        if (!wanted) return;
        if (b.accumulate && !given(mine)) raise(CHPL_ERR_INVALID, where, "accumulate wants %s to add to", name);
        t = given(mine) ? call.vector(name, mine, gt, b.n) : call.empty(b.n, gt);
        p = t.data_ptr();
    };
    rows_to("dx", PyObject_IsTrue(a[20]), a[24], dx, b.dx, b.lddx);
    if (join) {
        b.post = norm_of(call, "post", a + 8, b.n);
        b.gate = gate_of(call, a[5], b.tokens, b.n, &b.ldgate);
        const bool gate_wanted = given(a[5]) && PyObject_IsTrue(a[22]);
        if (b.post.kind || gate_wanted) b.y = call.matrix("y", a[4], call.type, b.tokens, b.n, &b.ldy).data_ptr();
        if (b.post.kind) b.post_stats = statistics(call, "post_stats", a[16], b.tokens);
        rows_to("dy", PyObject_IsTrue(a[21]), a[25], dy, b.dy, b.lddy);
        if (b.ldgate) rows_to("dgate", gate_wanted, a[26], dgate, b.dgate, b.lddgate);
        else sum_to("dgate", gate_wanted, a[26], dgate, b.dgate);
        sum_to("dpost.weight", params && b.post.kind, a[27], sums[0], b.dpost_weight);
        sum_to("dpost.bias", params && b.post.kind && b.post.bias, a[28], sums[1], b.dpost_bias);
    }
    sum_to(join ? "dpre.weight" : "dweight", params && b.pre.kind, a[29], sums[2], b.dpre_weight);
    sum_to(join ? "dpre.bias" : "dbias", params && b.pre.kind && b.pre.bias, a[30], sums[3], b.dpre_bias);
    size_t need = 0;
    check(chpl_norm_backward_worksize(&b, &need), "chpl_norm_backward_worksize");
    const Workspace work(call, a[31], need);
    check(chpl_norm_backward(call.stream(), &b, work.at, work.bytes), "chpl_norm_backward");
    PyObject* out = PyTuple_New(7);
    if (!out) throw python_error();
    at::Tensor* made[7] = {&dx, &dy, &dgate, &sums[0], &sums[1], &sums[2], &sums[3]};
    for (int i = 0; i < 7; ++i)
        PyTuple_SET_ITEM(out, i, !made[i]->defined() ? same_object(Py_None) : given(a[24 + i]) ? same_object(a[24 + i]) : wrap(std::move(*made[i])));
    return out;
    CHPL_PY_END
}

// ----------------------------------------------------------------------------
// microscaled 4-bit floating point
// ----------------------------------------------------------------------------
// the codes of a rows x cols matrix; bytes past the last group are not looked at
chpl_mx4 mx4_of(const Call& call, const char* name, PyObject* codes, PyObject* scales, int64_t rows, int64_t cols)
{
    chpl_mx4 c = {};
    char part[64];
    std::snprintf(part, sizeof(part), "%s.codes", name);
    c.codes = static_cast<uint8_t*>(call.matrix(part, codes, at::kByte, rows, (cols + kGroup - 1) / kGroup * (kGroup / 2), &c.ldc).data_ptr());
    std::snprintf(part, sizeof(part), "%s.scales", name);
    int64_t bytes = 0;
    check(chpl_mx4_scale_bytes(rows, cols, &bytes), "chpl_mx4_scale_bytes");
    c.scales = static_cast<uint8_t*>(call.vector(part, scales, at::kByte, bytes).data_ptr());
    return c;
}

int64_t columns(const char* where, PyObject* o)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    if (v < 0) raise(CHPL_ERR_INVALID, where, "%lld columns", v);
    return v;
}

// mx4_pack(x, codes, scales) -> (codes, scales)
PyObject* mx4_pack(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    CHPL_PY_BEGIN
    const char* where = "mx4.pack";
    arguments(where, n, 3);
    const at::Tensor& x = tensor(where, "x", a[0], 2);
    const int type = type_code(x.scalar_type());
    if (type < 0) raise(CHPL_ERR_INVALID, where, "x is %s: bfloat16, float16 or float32 is wanted", at::toString(x.scalar_type()));
    const int64_t ldx = row_distance(where, "x", x), rows = x.size(0), cols = x.size(1);
    const Call call(where, x);
    at::Tensor codes, scales;
    chpl_mx4 c = {};
    if (given(a[1])) {
        c = mx4_of(call, "out", a[1], a[2], rows, cols);
    } else {
        int64_t bytes = 0;
        check(chpl_mx4_scale_bytes(rows, cols, &bytes), "chpl_mx4_scale_bytes");
        c.ldc = (cols + kGroup - 1) / kGroup * (kGroup / 2);
        codes = call.empty(rows, c.ldc, at::kByte);
        scales = call.empty(bytes, at::kByte);
        c.codes = static_cast<uint8_t*>(codes.data_ptr());
        c.scales = static_cast<uint8_t*>(scales.data_ptr());
    }
    check(chpl_mx4_pack(call.stream(), type, rows, cols, x.data_ptr(), ldx, &c), "chpl_mx4_pack");
    if (given(a[1])) return PyTuple_Pack(2, a[1], a[2]);
    return Py_BuildValue("NN", wrap(std::move(codes)), wrap(std::move(scales)));
    CHPL_PY_END
}

// mx4_unpack(codes, scales, cols, dtype, out) -> x
PyObject* mx4_unpack(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    CHPL_PY_BEGIN
    const char* where = "mx4.unpack";
    arguments(where, n, 5);
    const at::Tensor& codes = tensor(where, "c.codes", a[0], 2);
    const int64_t rows = codes.size(0), cols = columns(where, a[2]);
    const Call call(where, codes);
    const chpl_mx4 c = mx4_of(call, "c", a[0], a[1], rows, cols);
    if (!THPDtype_Check(a[3])) raise(CHPL_ERR_INVALID, where, "dtype is not a torch.dtype");
    const at::ScalarType to = reinterpret_cast<THPDtype*>(a[3])->scalar_type;
    const int type = type_code(to);
    if (type < 0) raise(CHPL_ERR_INVALID, where, "%s: bfloat16, float16 or float32 is wanted", at::toString(to));
    int64_t ldx = cols;
    at::Tensor x = given(a[4]) ? call.matrix("out", a[4], to, rows, cols, &ldx) : call.empty(rows, cols, to);
    check(chpl_mx4_unpack(call.stream(), type, rows, cols, &c, x.data_ptr(), ldx), "chpl_mx4_unpack");
    return given(a[4]) ? same_object(a[4]) : wrap(std::move(x));
    CHPL_PY_END
}

// mx4_linear(x, x.codes, x.scales, x.cols, dtype, w.codes, w.scales, w.cols, bias, residual, act, out, work) -> Y
PyObject* mx4_linear(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    CHPL_PY_BEGIN
    const char* where = "mx4.linear";
    arguments(where, n, 13);
    const bool coded = !given(a[0]);
    const at::Tensor& x = coded ? tensor(where, "x.codes", a[1], 2) : tensor(where, "x", a[0], 2);
    const at::Tensor& w = tensor(where, "w.codes", a[5], 2);
    if (coded && !THPDtype_Check(a[4])) raise(CHPL_ERR_INVALID, where, "dtype is not a torch.dtype");
    Call call(where, x);
    if (coded) call.type = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
    chpl_mx4_fwd f = {};
    f.type = type_code(call.type);
    f.act = (int)number(a[10]);
    f.tokens = x.size(0);
    f.k = coded ? columns(where, a[3]) : x.size(1);
    f.n = w.size(0);
    const int64_t wk = columns(where, a[7]);
    if (wk != f.k) raise(CHPL_ERR_INVALID, where, "x has %lld features and w %lld", (long long)f.k, (long long)wk);
    if (coded) {
        f.x4 = mx4_of(call, "x", a[1], a[2], f.tokens, f.k);
    } else {
        f.x = x.data_ptr();
        f.ldx = row_distance(where, "x", x);
    }
    f.w4 = mx4_of(call, "w", a[5], a[6], f.n, f.k);
    if (given(a[8])) f.bias = call.vector("bias", a[8], call.type, f.n).data_ptr();
    if (given(a[9])) f.residual = call.matrix("residual", a[9], call.type, f.tokens, f.n, &f.ldr).data_ptr();
    f.ldy = f.n;
    at::Tensor y = given(a[11]) ? call.matrix("out", a[11], call.type, f.tokens, f.n, &f.ldy) : call.empty(f.tokens, f.n, call.type);
    f.y = y.data_ptr();
    size_t need = 0;
    check(chpl_mx4_linear_worksize(&f, &need), "chpl_mx4_linear_worksize");
    const Workspace work(call, a[12], need);
    check(chpl_mx4_linear(call.stream(), &f, work.at, work.bytes), "chpl_mx4_linear");
    return given(a[11]) ? same_object(a[11]) : wrap(std::move(y));
    CHPL_PY_END
}

#define CHPL_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CHPL_METHOD(ckpt8_pack), CHPL_METHOD(ckpt8_unpack), CHPL_METHOD(linear_forward),
                         CHPL_METHOD(linear_backward), CHPL_METHOD(norm_forward), CHPL_METHOD(norm_backward),
                         CHPL_METHOD(mx4_pack), CHPL_METHOD(mx4_unpack), CHPL_METHOD(mx4_linear), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch", "entry points of libchpl for a model's layers on torch tensors", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch(void) { return PyModule_Create(&module); }
