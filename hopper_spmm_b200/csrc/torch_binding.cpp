// The device-tensor product for Python: argument checks, output allocation, stream lookup and the call into the C
// ABI in one native function.  Through torch's Python attributes and ctypes the same steps take 8 us a call, more
// than the GPU needs for a 4096 x 4096 matrix at 1 % density.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#if __has_include(<ATen/cuda/EmptyTensor.h>)
#include <ATen/cuda/EmptyTensor.h>
#define HAS_EMPTY_CUDA 1
#endif
#include <ATen/record_function.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/b200_spmm.h"

namespace {

PyObject *refuse(const char *what) {
    PyErr_SetString(PyExc_ValueError, what);
    return nullptr;
}

// Other Python threads run while this exists.
struct ThreadsAllowed {
    PyThreadState *state = PyEval_SaveThread();
    ~ThreadsAllowed() { PyEval_RestoreThread(state); }
};

#ifdef HAS_EMPTY_CUDA
// torch's own, and not part of its interface: taken where it has the signature known here.
template <typename Type>
auto empty_direct(int, at::IntArrayRef sizes, Type type, at::Device device)
    -> decltype(at::Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt))) {
    return at::Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));
}
#endif
template <typename Type>
at::Tensor empty_direct(long, at::IntArrayRef, Type, at::Device) {
    return at::Tensor();
}

// A new CUDA tensor.  Through the dispatcher it is 1.2 of the 4.1 us that a small product takes the host, directly 0.9.  The
// dispatcher is left out only where nothing would happen in it but the allocation: no mode, tracer, transform or inference mode
// (the thread's keys are the default ones), no profiler or other observer of calls, and no fill that deterministic runs ask for.
at::Tensor new_cuda(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor &like) {
    const c10::impl::LocalDispatchKeySet keys = c10::impl::tls_local_dispatch_key_set();
    if (keys.included_ == c10::default_included_set && keys.excluded_ == c10::default_excluded_set && !at::hasCallbacks() &&
        !at::globalContext().deterministicAlgorithms()) {
        at::Tensor out = empty_direct(0, sizes, type, like.device());
        if (out.defined()) return out;
    }
    return at::empty(sizes, like.options().dtype(type).requires_grad(false));
}

// spmm(plan, is_f16, rows, cols, B, C or None, c_half, stream or None) -> C, or a status code that is not 0
// Any tensor accessor may throw: a sparse tensor has no strides, a tensor subclass may answer for sizes and strides in
// Python.  The macros turn whatever comes (a Python error among it) into the exception the caller sees.
PyObject *spmm(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 8) {
        PyErr_SetString(PyExc_TypeError, "spmm takes 8 arguments");
        return nullptr;
    }
    auto *plan = static_cast<b200spmm_plan_t *>(PyLong_AsVoidPtr(args[0]));
    const bool f16 = args[1] == Py_True, c_half = PyObject_IsTrue(args[6]) == 1;
    const int64_t rows = PyLong_AsLongLong(args[2]), cols = PyLong_AsLongLong(args[3]);
    if (PyErr_Occurred()) return nullptr;
    const char *bad_b = f16 ? "B must be a CUDA float16 tensor of shape [cols, n] with unit column stride"
                            : "B must be a CUDA float32 tensor of shape [cols, n] with unit column stride";
    if (!THPVariable_Check(args[4])) return refuse(bad_b);
    const at::Tensor &B = THPVariable_Unpack(args[4]);
    if (!B.is_cuda() || B.scalar_type() != (f16 ? at::kHalf : at::kFloat) || B.dim() != 2 || B.stride(1) != 1 || B.size(0) != cols)
        return refuse(bad_b);
    const int64_t n = B.size(1);
    const at::ScalarType c_type = c_half ? at::kHalf : at::kFloat;
    at::Tensor C;
    if (args[5] != Py_None) {
        if (!THPVariable_Check(args[5])) return refuse("C has the wrong shape, dtype or layout");
        C = THPVariable_Unpack(args[5]);
        if (!C.is_cuda() || C.scalar_type() != c_type || C.dim() != 2 || C.size(0) != rows || C.size(1) != n || C.stride(1) != 1)
            return refuse("C has the wrong shape, dtype or layout");
    }
    void *stream = nullptr;
    if (args[7] != Py_None) {
        stream = PyLong_AsVoidPtr(args[7]);
        if (PyErr_Occurred()) return nullptr;
    }
    if (args[5] == Py_None) C = new_cuda({rows, n}, c_type, B);
    if (args[7] == Py_None) stream = c10::cuda::getCurrentCUDAStream(B.get_device()).stream();
    const void *b = B.data_ptr();
    void *c = C.data_ptr();
    const int64_t ldb = B.stride(0), ldc = C.stride(0);
    int st;
    {  // the call waits for the device when a buffer of the plan grows, and for room when the stream's queue is full
        const ThreadsAllowed threads;
        st = b200spmm_spmm(plan, b, ldb, n, c, ldc, c_half ? B200SPMM_C_F16 : B200SPMM_C_F32, stream);
    }
    if (st != B200SPMM_OK) return PyLong_FromLong(st);
    if (args[5] != Py_None) {
        Py_INCREF(args[5]);
        return args[5];
    }
    return THPVariable_Wrap(std::move(C));
    END_HANDLE_TH_ERRORS
}

// ---- 4-bit matrices.  A matrix is (values, scales, tensor_scale, rows, cols, format) in the arguments.

// An argument that is a CUDA tensor, or null.  One whose numbers are to be negated when they are read (the imaginary part of a conjugate) is none.
const at::Tensor *cuda_tensor(PyObject *o) {
    if (!THPVariable_Check(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    return t.is_cuda() && !t.is_neg() ? &t : nullptr;
}

int type_code(at::ScalarType t) {
    return t == at::kFloat ? B200SPMM_T_F32 : t == at::kHalf ? B200SPMM_T_F16 : t == at::kBFloat16 ? B200SPMM_T_BF16 : -1;
}
at::ScalarType type_of(long code) { return code == B200SPMM_T_F16 ? at::kHalf : code == B200SPMM_T_BF16 ? at::kBFloat16 : at::kFloat; }

// A dense matrix with one dimension of neighbours: `transposed` where that is the first.
struct Dense {
    void *ptr;
    int64_t ld;
    bool transposed;
};
bool dense_of(const at::Tensor &t, Dense *d) {
    if (t.dim() != 2 || t.layout() != at::kStrided) return false;
    const int64_t r = t.size(0), c = t.size(1), sr = t.stride(0), sc = t.stride(1);
    if ((sc == 1 || c <= 1) && (r <= 1 || sr >= c)) *d = {nullptr, r <= 1 ? c : sr, false};
    else if ((sr == 1 || r <= 1) && (c <= 1 || sc >= r)) *d = {nullptr, c <= 1 ? r : sc, true};
    else return false;
    d->ptr = t.data_ptr();
    return true;
}

bool matrix_of(PyObject *const *args, b200spmm_fp4_t *m) {
    const at::Tensor *v = cuda_tensor(args[0]), *s = cuda_tensor(args[1]), *w = cuda_tensor(args[2]);
    if (!v || !s || !w || v->get_device() != s->get_device() || v->get_device() != w->get_device()) return false;
    m->values = v->data_ptr();
    m->scales = s->data_ptr();
    m->tensor_scale = static_cast<float *>(w->data_ptr());
    m->rows = PyLong_AsUnsignedLongLong(args[3]);
    m->cols = PyLong_AsUnsignedLongLong(args[4]);
    m->format = (int32_t)PyLong_AsLong(args[5]);
    m->device = (int32_t)v->get_device();
    return true;
}

// What X is quantised into, filled in on `stream`; the status.
int quantize_into(const at::Tensor &X, const Dense &x, const b200spmm_fp4_t *by_rows, const b200spmm_fp4_t *by_cols, const float *given) {
    const b200spmm_fp4_t &one = by_rows ? *by_rows : *by_cols;
    at::Tensor workspace;
    if (one.format == B200SPMM_NVFP4 && !given) {
        uint64_t bytes = 0;
        b200spmm_fp4_sizes(0, 0, one.format, nullptr, nullptr, nullptr, &bytes);
        workspace = new_cuda({(int64_t)bytes}, at::kByte, X);
    }
    void *ws = workspace.defined() ? workspace.data_ptr() : nullptr;
    void *stream = c10::cuda::getCurrentCUDAStream(X.get_device()).stream();
    const int code = type_code(X.scalar_type());
    const b200spmm_fp4_t *along = x.transposed ? by_cols : by_rows, *across = x.transposed ? by_rows : by_cols;  // the rows of X as they lie
    const ThreadsAllowed threads;
    if (along && across) return b200spmm_fp4_quantize_both(x.ptr, x.ld, code, given, along, across, ws, stream);
    return b200spmm_fp4_quantize(x.ptr, x.ld, code, across != nullptr, given, along ? along : across, ws, stream);
}

// X and a given scale (or None) as arguments; false with an error set where they will not do.
bool quantize_arguments(PyObject *const *args, const at::Tensor **X, Dense *x, const float **given) {
    *X = cuda_tensor(args[0]);
    if (!*X || type_code((*X)->scalar_type()) < 0 || !dense_of(**X, x)) {
        refuse("X must be a two-dimensional CUDA tensor of float32, float16 or bfloat16 with unit stride along rows or columns");
        return false;
    }
    *given = nullptr;
    if (args[1] != Py_None) {
        const at::Tensor *g = cuda_tensor(args[1]);
        if (!g || g->scalar_type() != at::kFloat || g->numel() != 1 || g->get_device() != (*X)->get_device()) {
            refuse("tensor_scale must be a float32 tensor of one element on X's device");
            return false;
        }
        *given = static_cast<const float *>(g->data_ptr());
    }
    return true;
}

// fp4_quantize(X, given scale or None, matrix, across) -> None or a status: into arrays that are there
PyObject *fp4_quantize(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 9) {
        PyErr_SetString(PyExc_TypeError, "fp4_quantize takes 9 arguments");
        return nullptr;
    }
    const at::Tensor *X;
    Dense x;
    const float *given;
    if (!quantize_arguments(args, &X, &x, &given)) return nullptr;
    b200spmm_fp4_t m{};
    const bool across = args[8] == Py_True;
    if (!matrix_of(args + 2, &m) || X->get_device() != m.device) return refuse("X and the matrix must be on the same CUDA device");
    if (PyErr_Occurred()) return nullptr;
    if (m.rows != (uint64_t)X->size(across ? 1 : 0) || m.cols != (uint64_t)X->size(across ? 0 : 1)) return refuse("the matrix does not have the shape of X");
    const int st = quantize_into(*X, x, across ? nullptr : &m, across ? &m : nullptr, given);
    if (st != B200SPMM_OK) return PyLong_FromLong(st);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// fp4_quantize_new(X, given scale or None, format, by rows, by columns) -> values, scales, scale of either (one after the other), or a status
PyObject *fp4_quantize_new(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 5) {
        PyErr_SetString(PyExc_TypeError, "fp4_quantize_new takes 5 arguments");
        return nullptr;
    }
    const at::Tensor *X;
    Dense x;
    const float *given;
    if (!quantize_arguments(args, &X, &x, &given)) return nullptr;
    const long format = PyLong_AsLong(args[2]);
    if (PyErr_Occurred()) return nullptr;
    const bool want[2] = {args[3] == Py_True, args[4] == Py_True};
    at::Tensor made[2][3];
    b200spmm_fp4_t m[2] = {};
    for (int i = 0; i < 2; ++i) {
        if (!want[i]) continue;
        m[i].rows = (uint64_t)X->size(i);
        m[i].cols = (uint64_t)X->size(1 - i);
        m[i].format = (int32_t)format;
        m[i].device = (int32_t)X->get_device();
        uint64_t pitch = 0, scales = 0;
        const int st = b200spmm_fp4_sizes(m[i].rows, m[i].cols, (int)format, &pitch, nullptr, &scales, nullptr);
        if (st != B200SPMM_OK) return PyLong_FromLong(st);
        made[i][0] = new_cuda({(int64_t)m[i].rows, (int64_t)pitch}, at::kByte, *X);
        made[i][1] = new_cuda({(int64_t)scales}, at::kByte, *X);
        made[i][2] = new_cuda({1}, at::kFloat, *X);
        m[i].values = made[i][0].data_ptr();
        m[i].scales = made[i][1].data_ptr();
        m[i].tensor_scale = static_cast<float *>(made[i][2].data_ptr());
    }
    const int st = quantize_into(*X, x, want[0] ? &m[0] : nullptr, want[1] ? &m[1] : nullptr, given);
    if (st != B200SPMM_OK) return PyLong_FromLong(st);
    PyObject *out = PyTuple_New(want[0] && want[1] ? 6 : 3);
    if (!out) return nullptr;
    Py_ssize_t at = 0;
    for (int i = 0; i < 2; ++i)
        for (int j = 0; want[i] && j < 3; ++j) PyTuple_SET_ITEM(out, at++, THPVariable_Wrap(std::move(made[i][j])));
    return out;
    END_HANDLE_TH_ERRORS
}

// C for a product of `rows` x `n`: the caller's, or a new one.  Null with an error set where it does not fit.
bool output_of(PyObject *arg, int64_t rows, int64_t n, long type, const at::Tensor &like, at::Tensor *C, Dense *c) {
    const char *bad = "C has the wrong shape, dtype, device or layout";
    if (arg == Py_None) {
        *C = new_cuda({rows, n}, type_of(type), like);
    } else {
        const at::Tensor *t = cuda_tensor(arg);
        if (!t || t->scalar_type() != type_of(type) || t->dim() != 2 || t->size(0) != rows || t->size(1) != n || t->get_device() != like.get_device()) {
            refuse(bad);
            return false;
        }
        *C = *t;
    }
    if (!dense_of(*C, c)) {
        refuse(bad);
        return false;
    }
    return true;
}

// The workspace of a product of `a` with n columns; nothing where it needs none (or cannot be asked: the product will say why).
at::Tensor product_workspace(const b200spmm_fp4_t &a, const Dense *b, int64_t n, const at::Tensor &like, uint64_t *bytes) {
    *bytes = 0;
    if (b200spmm_fp4_product_workspace(&a, b ? b->ptr : nullptr, b ? b->ld : 0, n, b && b->transposed, bytes) != B200SPMM_OK || *bytes == 0) return at::Tensor();
    return new_cuda({(int64_t)*bytes}, at::kByte, like);
}

PyObject *result_of(int st, PyObject *arg, at::Tensor &&C) {
    if (st != B200SPMM_OK) return PyLong_FromLong(st);
    if (arg != Py_None) {
        Py_INCREF(arg);
        return arg;
    }
    return THPVariable_Wrap(std::move(C));
}

// fp4_dequantize(matrix, X or None, type) -> X or a status
PyObject *fp4_dequantize(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    b200spmm_fp4_t a{};
    if (n_args != 8 || !matrix_of(args, &a)) return refuse("the matrix must be on one CUDA device");
    const long type = PyLong_AsLong(args[7]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor &like = *cuda_tensor(args[0]);
    at::Tensor X;
    Dense x;
    if (!output_of(args[6], (int64_t)a.rows, (int64_t)a.cols, type, like, &X, &x)) return nullptr;
    if (x.transposed) return refuse("the values are written row by row: unit stride along the rows");
    void *stream = c10::cuda::getCurrentCUDAStream(like.get_device()).stream();
    int st;
    {
        const ThreadsAllowed threads;
        st = b200spmm_fp4_dequantize(&a, x.ptr, x.ld, (int)type, stream);
    }
    return result_of(st, args[6], std::move(X));
    END_HANDLE_TH_ERRORS
}

// fp4_product(matrix, matrix, C or None, type) -> C or a status
PyObject *fp4_product(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    b200spmm_fp4_t a{}, b{};
    if (n_args != 14 || !matrix_of(args, &a) || !matrix_of(args + 6, &b)) return refuse("the matrices must be on one CUDA device");
    const long type = PyLong_AsLong(args[13]);
    if (PyErr_Occurred()) return nullptr;
    if (a.device != b.device) return refuse("the matrices must be on one CUDA device");
    if (a.cols != b.cols) return refuse("the matrices must have the same number of columns");
    const at::Tensor &like = *cuda_tensor(args[0]);
    at::Tensor C;
    Dense c;
    if (!output_of(args[12], (int64_t)a.rows, (int64_t)b.rows, type, like, &C, &c)) return nullptr;
    void *stream = c10::cuda::getCurrentCUDAStream(like.get_device()).stream();
    uint64_t bytes;
    const at::Tensor workspace = product_workspace(a, nullptr, (int64_t)b.rows, like, &bytes);
    void *ws = workspace.defined() ? workspace.data_ptr() : nullptr;
    int st;
    {
        const ThreadsAllowed threads;
        st = b200spmm_fp4_product(&a, &b, c.ptr, c.ld, (int)type, c.transposed, ws, bytes, stream);
    }
    return result_of(st, args[12], std::move(C));
    END_HANDLE_TH_ERRORS
}

// fp4_dense_product(matrix, B, C or None, type) -> C or a status
PyObject *fp4_dense_product(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    b200spmm_fp4_t a{};
    if (n_args != 9 || !matrix_of(args, &a)) return refuse("the matrix must be on one CUDA device");
    const long type = PyLong_AsLong(args[8]);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor *B = cuda_tensor(args[6]);
    const int b_type = B ? type_code(B->scalar_type()) : -1;
    Dense b;
    if (!B || b_type < 0 || b_type == B200SPMM_T_F32 || !dense_of(*B, &b) || (uint64_t)B->size(0) != a.cols || B->get_device() != a.device)
        return refuse("B must be a CUDA float16 or bfloat16 tensor of shape [cols, n] on the matrix's device with unit stride along rows or columns");
    at::Tensor C;
    Dense c;
    if (!output_of(args[7], (int64_t)a.rows, B->size(1), type, *B, &C, &c)) return nullptr;
    void *stream = c10::cuda::getCurrentCUDAStream(B->get_device()).stream();
    const int64_t n = B->size(1);
    uint64_t bytes;
    const at::Tensor workspace = product_workspace(a, &b, n, *B, &bytes);
    void *ws = workspace.defined() ? workspace.data_ptr() : nullptr;
    int st;
    {
        const ThreadsAllowed threads;
        st = b200spmm_fp4_dense_product(&a, b.ptr, b.ld, n, b_type, b.transposed, c.ptr, c.ld, (int)type, c.transposed, ws, bytes, stream);
    }
    return result_of(st, args[7], std::move(C));
    END_HANDLE_TH_ERRORS
}

template <PyObject *(*kFn)(PyObject *, PyObject *const *, Py_ssize_t)>
PyCFunction fast() { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kFn)); }

PyMethodDef methods[] = {{"spmm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(spmm)), METH_FASTCALL, nullptr},
                         {"fp4_quantize", fast<fp4_quantize>(), METH_FASTCALL, nullptr},
                         {"fp4_quantize_new", fast<fp4_quantize_new>(), METH_FASTCALL, nullptr},
                         {"fp4_dequantize", fast<fp4_dequantize>(), METH_FASTCALL, nullptr},
                         {"fp4_product", fast<fp4_product>(), METH_FASTCALL, nullptr},
                         {"fp4_dense_product", fast<fp4_dense_product>(), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding(void) { return PyModule_Create(&module); }
