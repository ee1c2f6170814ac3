/* bind.cpp -- the call path of ops.py's int8 step in C++: torch tensors to RadArgs, resolution, launch. What the
 * ctypes harness of plugin.py does for a row (operands by schema position, the row with the highest priority whose
 * constraints hold, its launch pointer on the current stream), at 4 us a call on the host, the launch included (6 to 8 where
 * ops.py makes the results), instead of 97: a decode step's kernels take 2 to 25 us each. Nothing is computed here, and
 * nothing of a call is remembered.
 */
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cstring>
#include <vector>
#include "rad_abi.h"
#include "r3d_b200.h"

namespace {

constexpr int kMaxTensors = 12, kMaxParams = 12;

bool type_of(at::ScalarType t, uint32_t* out) {
    switch (t) {
        case at::kFloat:    *out = RAD_F32; return true;
        case at::kBFloat16: *out = RAD_BF16; return true;
        case at::kChar:     *out = RAD_I8; return true;
        case at::kInt:      *out = RAD_I32; return true;
        default:            return false;
    }
}

/* a constraint on a key the call does not carry does not hold (src/r3d_rows.cpp:1105-1110 of libr3d) */
bool holds(const RadConstraint& c, const RadParam* p, int n) {
    for (int i = 0; i < n; ++i) {
        if (strcmp(p[i].key, c.key) != 0) continue;
        if (c.op == RAD_C_IN) {
            if (p[i].kind != RAD_PK_STR || !c.sval) return false;
            const size_t len = strlen(p[i].sval);
            for (const char* at = c.sval; (at = strstr(at, p[i].sval)) != nullptr && len; ++at)
                if ((at == c.sval || at[-1] == ' ') && (at[len] == ' ' || at[len] == 0)) return true;
            return false;
        }
        if (p[i].kind != RAD_PK_INT) return false;
        const long long v = p[i].ival;
        return c.op == RAD_C_EQ ? v == c.ival : c.op == RAD_C_LE ? v <= c.ival : c.op == RAD_C_GE ? v >= c.ival
             : c.op == RAD_C_DIV ? c.ival != 0 && v % c.ival == 0 : false;
    }
    return false;
}

/* the loader's rows and behind them the extension rows. Both tables are fixed for the process, and walking the loader's by
 * index takes 3 us: they are walked once */
const std::vector<const RadKernelInfo*>& all_rows() {
    static const std::vector<const RadKernelInfo*> all = [] {
        std::vector<const RadKernelInfo*> v;
        for (int i = 0; const RadKernelInfo* k = rad_kernel_at(i); ++i) v.push_back(k);
        for (int i = 0; const RadKernelInfo* k = r3d_b200_ext_kernel_at(i); ++i) v.push_back(k);
        return v;
    }();
    return all;
}

/* highest priority, the first declared among equals */
const RadKernelInfo* resolve(const char* op, const RadParam* p, int n) {
    const RadKernelInfo* best = nullptr;
    for (const RadKernelInfo* k : all_rows()) {
        if (strcmp(k->op, op) != 0 || (best && k->priority <= best->priority)) continue;
        bool fits = true;
        for (int i = 0; i < k->n_constraints && fits; ++i) fits = holds(k->constraints[i], p, n);
        if (fits) best = k;
    }
    return best;
}

/* on the operands' device and its current stream; torch's errors become the device status */
int launch_on(int dev, const RadKernelInfo* row, const RadArgs& a) noexcept {
    try {
        const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
        return row->launch(&a, (RadStream)c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream());
    } catch (...) {
        return RAD_E_DEVICE;
    }
}

/* issue(op, ((key, value), ...), tensor or None, ...) -> None, or (row name or None, status) of a call not taken */
PyObject* issue_or_throw(PyObject* const* args, Py_ssize_t nargs) {
    if (nargs < 3 || nargs - 2 > kMaxTensors || !PyTuple_Check(args[1]) || PyTuple_GET_SIZE(args[1]) > kMaxParams) {
        PyErr_SetString(PyExc_TypeError, "issue(op, params, tensor or None, ...)");
        return nullptr;
    }
    const char* op = PyUnicode_AsUTF8(args[0]);
    if (!op) return nullptr;
    RadParam p[kMaxParams];
    const int np = (int)PyTuple_GET_SIZE(args[1]);
    memset(p, 0, sizeof p);
    for (int i = 0; i < np; ++i) {
        PyObject* kv = PyTuple_GET_ITEM(args[1], i);
        if (!PyTuple_Check(kv) || PyTuple_GET_SIZE(kv) != 2) { PyErr_SetString(PyExc_TypeError, "params are (key, value) pairs"); return nullptr; }
        PyObject* v = PyTuple_GET_ITEM(kv, 1);
        p[i].key = PyUnicode_AsUTF8(PyTuple_GET_ITEM(kv, 0));
        if (PyUnicode_Check(v)) { p[i].kind = RAD_PK_STR; p[i].sval = PyUnicode_AsUTF8(v); }
        else if (PyFloat_Check(v)) { p[i].kind = RAD_PK_F64; p[i].dval = PyFloat_AS_DOUBLE(v); }
        else { p[i].kind = RAD_PK_INT; p[i].ival = PyLong_AsLongLong(v); }
        if (!p[i].key || PyErr_Occurred()) return nullptr;
    }
    RadTensor t[kMaxTensors];
    memset(t, 0, sizeof t);
    int dev = -1;
    for (int i = 0; i < (int)nargs - 2; ++i) {
        PyObject* o = args[i + 2];
        t[i].dtype = RAD_F32;
        if (o == Py_None) continue;
        if (!THPVariable_Check(o)) { PyErr_Format(PyExc_TypeError, "%s: operands are tensors, got %s", op, Py_TYPE(o)->tp_name); return nullptr; }
        const at::ScalarType type = THPVariable_Unpack(o).scalar_type();
        if (!type_of(type, &t[i].dtype)) { PyErr_Format(PyExc_TypeError, "%s: no %s operands", op, c10::toString(type)); return nullptr; }
    }
    for (int i = 0; i < (int)nargs - 2; ++i) {
        if (args[i + 2] == Py_None) continue;
        const at::Tensor& x = THPVariable_Unpack(args[i + 2]);
        if (!x.is_cuda() || (dev >= 0 && x.get_device() != dev)) { PyErr_Format(PyExc_ValueError, "%s: operands on one CUDA device are needed", op); return nullptr; }
        if (x.dim() > RAD_MAX_RANK) { PyErr_Format(PyExc_ValueError, "%s: at most %d dimensions", op, RAD_MAX_RANK); return nullptr; }
        dev = x.get_device();
        t[i].data = x.data_ptr();
        t[i].rank = (uint32_t)x.dim();
        for (int d = 0; d < (int)x.dim(); ++d) { t[i].shape[d] = x.size(d); t[i].stride[d] = x.stride(d); }
    }
    if (dev < 0) { PyErr_Format(PyExc_ValueError, "%s: operands on one CUDA device are needed", op); return nullptr; }
    const RadKernelInfo* row = resolve(op, p, np);
    if (!row) return Py_BuildValue("(Oi)", Py_None, (int)RAD_E_UNSUPPORTED);
    RadArgs a;
    memset(&a, 0, sizeof a);
    a.t = t; a.n_t = (int)nargs - 2; a.p = p; a.n_p = np;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = launch_on(dev, row, a);
    Py_END_ALLOW_THREADS
    if (rc != RAD_OK) return Py_BuildValue("(si)", row->name, rc);
    Py_RETURN_NONE;
}

PyObject* issue(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    try {
        return issue_or_throw(args, nargs);
    } catch (const std::exception& e) {                /* a tensor without storage, say */
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

at::Tensor rows_of(const at::Tensor& x, long long n, at::ScalarType type) {
    int64_t size[RAD_MAX_RANK];
    const int lead = (int)x.dim() - 1;
    for (int d = 0; d < lead; ++d) size[d] = x.size(d);
    size[lead] = n;
    return at::empty(at::IntArrayRef(size, (size_t)(n < 0 ? lead : lead + 1)), x.options().dtype(type).requires_grad(false));
}

/* rows(x, n, type): a new tensor of x's leading dimensions and n columns (n < 0: no columns) on x's device.
 * type: 0 f32, 1 bf16, 2 int8, 3 int32 */
PyObject* rows(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 3 || !THPVariable_Check(args[0])) { PyErr_SetString(PyExc_TypeError, "rows(tensor, n, type)"); return nullptr; }
    const long long n = PyLong_AsLongLong(args[1]);
    const long type = PyLong_AsLong(args[2]);
    if (PyErr_Occurred()) return nullptr;
    static const at::ScalarType types[4] = {at::kFloat, at::kBFloat16, at::kChar, at::kInt};
    const at::Tensor& x = THPVariable_Unpack(args[0]);
    if (type < 0 || type > 3 || x.dim() < 1 || x.dim() > RAD_MAX_RANK) { PyErr_SetString(PyExc_ValueError, "1 to 8 dimensions are needed"); return nullptr; }
    try {
        return THPVariable_Wrap(rows_of(x, n, types[type]));
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

/* codes(x, n): new int8 codes [..., n] and f32 scales [..., 1] for x's rows */
PyObject* codes(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 2 || !THPVariable_Check(args[0])) { PyErr_SetString(PyExc_TypeError, "codes(tensor, n)"); return nullptr; }
    const long long n = PyLong_AsLongLong(args[1]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor& x = THPVariable_Unpack(args[0]);
    if (n < 0 || x.dim() < 1 || x.dim() > RAD_MAX_RANK) { PyErr_SetString(PyExc_ValueError, "1 to 8 dimensions are needed"); return nullptr; }
    PyObject* q = nullptr;
    try {
        q = THPVariable_Wrap(rows_of(x, n, at::kChar));
        PyObject* s = q ? THPVariable_Wrap(rows_of(x, 1, at::kFloat)) : nullptr;
        PyObject* both = s ? PyTuple_New(2) : nullptr;
        if (!both) { Py_XDECREF(q); Py_XDECREF(s); return nullptr; }
        PyTuple_SET_ITEM(both, 0, q);
        PyTuple_SET_ITEM(both, 1, s);
        return both;
    } catch (const std::exception& e) {
        Py_XDECREF(q);
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyMethodDef kMethods[] = {
    {"issue", (PyCFunction)(void (*)(void))issue, METH_FASTCALL, "one call of an op through its row"},
    {"codes", (PyCFunction)(void (*)(void))codes, METH_FASTCALL, "new codes and scales for a tensor's rows"},
    {"rows", (PyCFunction)(void (*)(void))rows, METH_FASTCALL, "a new tensor of another's rows"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

} /* namespace */

PyMODINIT_FUNC PyInit__bind(void) { return PyModule_Create(&kModule); }
