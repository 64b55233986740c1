// Python bindings of the linear-layer entry points for torch tensors: the module
// chpl_b200._torch, which chpl_b200/ckpt8.py and linear.py call.
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
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/autograd/python_variable.h>

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
    at::Tensor empty(int64_t rows, int64_t cols, at::ScalarType t) const
    {
        return at::empty({rows, cols}, at::TensorOptions().dtype(t).device(device));
    }
    at::Tensor empty(int64_t n, at::ScalarType t) const { return at::empty({n}, at::TensorOptions().dtype(t).device(device)); }

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

#define CHPL_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CHPL_METHOD(ckpt8_pack), CHPL_METHOD(ckpt8_unpack), CHPL_METHOD(linear_forward),
                         CHPL_METHOD(linear_backward), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch", "linear-layer entry points of libchpl for torch tensors", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch(void) { return PyModule_Create(&module); }
