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
#include <c10/core/AutogradState.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAStream.h>
#include <ATen/core/grad_mode.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <memory>
#include <vector>

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

// Autograd is told that a caller's tensor has other values now: what saved it for a backward pass must not use it any more.
void written(const at::Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void written(PyObject *arg) {
    if (arg != Py_None) written(THPVariable_Unpack(arg));
}

PyObject *result_of(int st, PyObject *arg, at::Tensor &&C) {
    if (st != B200SPMM_OK) return PyLong_FromLong(st);
    if (arg != Py_None) {
        written(C);
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

// ---- around weights in few bits

// Whether a gradient would be lost: the tensor wants one and gradients are recorded, or it has a tangent and those are taken along.
bool wants_gradient(const at::Tensor &t) {
    return (t.requires_grad() && at::GradMode::is_enabled()) || (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode());
}
constexpr const char *kNoGradient = "there is no backward pass, nor a forward-mode one: call it under torch.no_grad(), or with tensors that require no gradient and have no tangent";

// Rows of neighbours: the address and the distance of rows, in elements.
struct Rows {
    void *ptr;
    int64_t ld;
};
bool rows_of(const at::Tensor &t, Rows *r) {
    if (t.dim() != 2 || t.layout() != at::kStrided) return false;
    const int64_t n = t.size(0), c = t.size(1);
    if ((c > 1 && t.stride(1) != 1) || (n > 1 && t.stride(0) < c)) return false;
    *r = {t.data_ptr(), n <= 1 ? c : t.stride(0)};
    return true;
}

PyObject *three(PyObject *a, PyObject *b, PyObject *c) {
    PyObject *out = a && b && c ? PyTuple_New(3) : nullptr;
    if (!out) {
        Py_XDECREF(a);
        Py_XDECREF(b);
        Py_XDECREF(c);
        return nullptr;
    }
    PyTuple_SET_ITEM(out, 0, a);
    PyTuple_SET_ITEM(out, 1, b);
    PyTuple_SET_ITEM(out, 2, c);
    return out;
}
PyObject *again(PyObject *o) {
    Py_INCREF(o);
    return o;
}

// rms_norm(X, weight or None, eps, residual or None, sum or None, out or None, scales or None, out's type, group) -> (out, scales or None, sum or
// None), the first of them a status where it is a number
PyObject *rms_norm(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 9) {
        PyErr_SetString(PyExc_TypeError, "rms_norm takes 9 arguments");
        return nullptr;
    }
    b200spmm_rms_norm_t p{};
    const at::Tensor *X = cuda_tensor(args[0]);
    Rows x, r, o, h;
    if (!X || type_code(X->scalar_type()) < 0 || !rows_of(*X, &x))
        return refuse("X must be a two-dimensional CUDA tensor of float32, float16 or bfloat16 with unit stride along its rows");
    p.eps = (float)PyFloat_AsDouble(args[2]);
    const long type = PyLong_AsLong(args[7]), group = PyLong_AsLong(args[8]);
    if (PyErr_Occurred()) return nullptr;
    if (!(p.eps >= 0.f)) return refuse("eps must not be negative");
    const bool e4m3 = type == B200SPMM_T_E4M3;
    const int64_t rows = X->size(0), cols = X->size(1);
    bool lost = wants_gradient(*X);
    auto beside = [&](const at::Tensor *t) { return t && t->get_device() == X->get_device(); };
    if (args[1] != Py_None) {
        const at::Tensor *w = cuda_tensor(args[1]);
        if (!beside(w) || type_code(w->scalar_type()) < 0 || w->layout() != at::kStrided || w->dim() != 1 || w->size(0) != cols || (cols > 1 && w->stride(0) != 1))
            return refuse("weight must be a contiguous tensor of X's number of columns, float32, float16 or bfloat16, on X's device");
        lost = lost || wants_gradient(*w);
        p.weight = w->data_ptr();
        p.w_dtype = type_code(w->scalar_type());
    }
    auto like_x = [&](const at::Tensor *t, at::ScalarType kind, Rows *at) {
        return beside(t) && t->scalar_type() == kind && t->dim() == 2 && t->size(0) == rows && t->size(1) == cols && rows_of(*t, at);
    };
    at::Tensor sum, out, scales;
    if (args[3] != Py_None) {
        const at::Tensor *t = cuda_tensor(args[3]);
        if (!t || (t->scalar_type() != X->scalar_type() && t->scalar_type() != at::kFloat) || !like_x(t, t->scalar_type(), &r))
            return refuse("residual must be a tensor of X's shape, on X's device, of X's type or float32, with unit stride along its rows");
        lost = lost || wants_gradient(*t);
        p.residual = r.ptr;
        p.ldr = r.ld;
        p.r_dtype = type_code(t->scalar_type());
        if (args[4] != Py_None) {
            const at::Tensor *s = cuda_tensor(args[4]);
            if (!like_x(s, t->scalar_type(), &h)) return refuse("sum_out must be a tensor like residual with unit stride along its rows");
            lost = lost || wants_gradient(*s);
        }
    } else if (args[4] != Py_None) {
        return refuse("sum_out is for a call with a residual");
    }
    const at::ScalarType out_type = e4m3 ? at::kFloat8_e4m3fn : type_of(type);
    const int64_t groups = group ? (cols + group - 1) / group : 1;
    if (args[5] != Py_None) {
        const at::Tensor *t = cuda_tensor(args[5]), *s = args[6] == Py_None ? nullptr : cuda_tensor(args[6]);
        if (!like_x(t, out_type, &o) || (e4m3 && (!beside(s) || s->scalar_type() != at::kFloat || s->dim() != 2 || s->size(0) != rows || s->size(1) != groups || !s->is_contiguous())))
            return refuse("out has the wrong shape, type, device or layout");
        lost = lost || wants_gradient(*t);
        if (e4m3) p.scales = static_cast<float *>(s->data_ptr());
    }
    if (lost) return refuse(kNoGradient);
    if (args[5] == Py_None) {
        out = new_cuda({rows, cols}, out_type, *X);
        o = {out.data_ptr(), cols};
        if (e4m3) {
            scales = new_cuda({rows, groups}, at::kFloat, *X);
            p.scales = static_cast<float *>(scales.data_ptr());
        }
    }
    if (args[3] != Py_None && args[4] == Py_None) {  // (an empty tensor has no address)
        sum = new_cuda({rows, cols}, p.r_dtype == B200SPMM_T_F32 ? at::kFloat : X->scalar_type(), *X);
        h = {sum.data_ptr(), cols};
    }
    p.rows = (uint64_t)rows;
    p.cols = (uint64_t)cols;
    p.x_dtype = type_code(X->scalar_type());
    p.out_dtype = (int32_t)type;
    p.group = (int32_t)group;
    p.device = (int32_t)X->get_device();
    p.x = x.ptr;
    p.ldx = x.ld;
    p.out = o.ptr;
    p.ldo = o.ld;
    if (args[3] != Py_None) {
        p.sum = h.ptr;
        p.lds = h.ld;
    }
    void *stream = c10::cuda::getCurrentCUDAStream(X->get_device()).stream();
    int st;
    {
        const ThreadsAllowed threads;
        st = b200spmm_rms_norm(&p, stream);
    }
    if (st != B200SPMM_OK) return three(PyLong_FromLong(st), again(Py_None), again(Py_None));
    for (int i : {4, 5}) written(args[i]);
    if (e4m3 && args[5] != Py_None) written(args[6]);
    PyObject *a = out.defined() ? THPVariable_Wrap(std::move(out)) : again(args[5]);
    PyObject *b = scales.defined() ? THPVariable_Wrap(std::move(scales)) : again(Py_None);
    PyObject *c = sum.defined() ? THPVariable_Wrap(std::move(sum)) : again(args[4]);
    return three(a, b, c);
    END_HANDLE_TH_ERRORS
}

// A tensor whose address a capsule keeps.  What it was stays alive with it, so that nothing else can come to lie there; a call refuses one that has become another since
// (`t.data = ...`, a module's `.to()`, `resize_`), or that has come to want a gradient.
struct Held {
    at::Tensor now, was;
    const void *at;
    explicit Held(const at::Tensor &t) : now(t), was(t.detach()), at(t.data_ptr()) {}
    bool same() const { return now.data_ptr() == at && now.scalar_type() == was.scalar_type() && now.sizes() == was.sizes() && now.strides() == was.strides(); }
};
const char *fault_of(const std::vector<Held> &held) {
    for (const Held &h : held) {
        if (!h.same()) return "a tensor that was kept has another storage, type or shape now: make the matrix or the layer anew";
        if (wants_gradient(h.now)) return kNoGradient;
    }
    return nullptr;
}

// A matrix of 4-bit integers: what the C ABI gets of it, behind a capsule.
constexpr const char *kInt4 = "b200spmm_int4_t";
struct Int4 {
    b200spmm_int4_t m{};
    std::vector<Held> held;
};
void free_int4(PyObject *capsule) { delete static_cast<Int4 *>(PyCapsule_GetPointer(capsule, kInt4)); }

// int4_matrix(values, scales, zeros or None, rows, cols, group) -> capsule
PyObject *int4_matrix(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 6) {
        PyErr_SetString(PyExc_TypeError, "int4_matrix takes 6 arguments");
        return nullptr;
    }
    const int64_t rows = PyLong_AsLongLong(args[3]), cols = PyLong_AsLongLong(args[4]), group = PyLong_AsLongLong(args[5]);
    if (PyErr_Occurred()) return nullptr;
    if (rows < 0 || cols < 0 || rows > 0x7FFFFFFF - 256 || cols > 0x7FFFFFFF - 512) return refuse("rows and cols must lie between 0 and 2^31");
    if (group != 0 && (group < 32 || group > (1 << 30) || (group & (group - 1)) != 0)) return refuse("group must be None (a whole row) or a power of two from 32 on");
    auto tensor = [&](PyObject *o, int64_t a, int64_t b) -> const at::Tensor * {
        if (!THPVariable_Check(o)) return nullptr;
        const at::Tensor &t = THPVariable_Unpack(o);
        return t.layout() == at::kStrided && t.dim() == 2 && t.size(0) == a && t.size(1) == b && t.is_contiguous() && !t.is_neg() ? &t : nullptr;
    };
    const int64_t groups = group ? (cols + group - 1) / group : 1;
    const at::Tensor *v = tensor(args[0], rows, (cols + 31) / 32 * 16), *s = tensor(args[1], groups, rows), *z = args[2] == Py_None ? nullptr : tensor(args[2], groups, rows);
    if (!v || v->scalar_type() != at::kByte) return refuse("values must be a contiguous uint8 tensor [rows, 16 for every 32 columns begun]");
    if (!s || (s->scalar_type() != at::kHalf && s->scalar_type() != at::kBFloat16)) return refuse("scales must be a contiguous float16 or bfloat16 tensor [groups of a row, rows]");
    if (args[2] != Py_None && (!z || z->scalar_type() != at::kByte)) return refuse("zeros must be a contiguous uint8 tensor [groups of a row, rows]");
    if (wants_gradient(*s)) return refuse(kNoGradient);
    if (s->device() != v->device() || (z && z->device() != v->device())) return refuse("values, scales and zeros must be on one device");
    if (!v->is_cuda()) return refuse("values, scales and zeros must be on a CUDA device");
    auto made = std::make_unique<Int4>();
    b200spmm_int4_t *m = &made->m;
    m->rows = (uint64_t)rows;
    m->cols = (uint64_t)cols;
    m->group = (int32_t)group;
    m->scale_dtype = type_code(s->scalar_type());
    m->device = (int32_t)v->get_device();
    m->values = v->data_ptr();
    m->scales = s->data_ptr();
    m->zeros = z ? static_cast<const uint8_t *>(z->data_ptr()) : nullptr;
    made->held = {Held(*v), Held(*s)};
    if (z) made->held.emplace_back(*z);
    PyObject *out = PyCapsule_New(made.get(), kInt4, free_int4);
    if (out) made.release();
    return out;
    END_HANDLE_TH_ERRORS
}

// int4_product(capsule, B or values, their scales or None, group, C or None, type, tokens first) -> C or a status.  Tokens first: B is [n, cols] and C
// [n, rows], else [cols, n] and [rows, n]; 8-bit B always [n, cols].
PyObject *int4_product(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 7) {
        PyErr_SetString(PyExc_TypeError, "int4_product takes 7 arguments");
        return nullptr;
    }
    const auto *matrix = static_cast<const Int4 *>(PyCapsule_GetPointer(args[0], kInt4));
    const long group = PyLong_AsLong(args[3]), type = PyLong_AsLong(args[5]);
    if (PyErr_Occurred()) return nullptr;
    const b200spmm_int4_t *a = &matrix->m;
    if (const char *fault = fault_of(matrix->held)) return refuse(fault);
    const bool first = args[6] == Py_True, eights = args[2] != Py_None;
    const at::Tensor *B = cuda_tensor(args[1]), *s = eights ? cuda_tensor(args[2]) : nullptr;
    Dense b;
    const bool lies_first = first || eights;
    if (!B || B->scalar_type() != (eights ? at::kFloat8_e4m3fn : B->scalar_type() == at::kHalf ? at::kHalf : at::kBFloat16) || !dense_of(*B, &b) || (eights && b.transposed && B->size(0) > 1) ||
        B->size(lies_first ? 1 : 0) != (int64_t)a->cols || B->get_device() != a->device)
        return refuse(eights ? "the 8-bit matrix must have the matrix's columns, on its device, with unit stride along its rows"
                             : first ? "X must be a CUDA float16 or bfloat16 tensor of shape [n, cols] on the matrix's device with unit stride along rows or columns"
                                     : "B must be a CUDA float16 or bfloat16 tensor of shape [cols, n] on the matrix's device with unit stride along rows or columns");
    const int64_t n = B->size(lies_first ? 0 : 1);
    if (eights && (!s || s->get_device() != a->device || s->scalar_type() != at::kFloat || (group != 0 && group != 32 && group != 64 && group != 128) || s->dim() != 2 || s->size(0) != n ||
                   s->size(1) != (group ? ((int64_t)a->cols + group - 1) / group : 1) || !s->is_contiguous()))
        return refuse("the 8-bit matrix's scales must be contiguous float32, [n, groups of a row], on the matrix's device");
    if (wants_gradient(*B) || (s && wants_gradient(*s))) return refuse(kNoGradient);
    if (eights && b.transposed) b = {b.ptr, (int64_t)a->cols, false};  // (one row)
    at::Tensor C;
    Dense c;
    if (!output_of(args[4], first ? n : (int64_t)a->rows, first ? (int64_t)a->rows : n, type, *B, &C, &c)) return nullptr;
    if (wants_gradient(C)) return refuse(kNoGradient);
    void *stream = c10::cuda::getCurrentCUDAStream(B->get_device()).stream();
    int st;
    {
        const ThreadsAllowed threads;
        st = b200spmm_int4_product(a, b.ptr, b.ld, n, eights ? B200SPMM_T_E4M3 : type_code(B->scalar_type()), lies_first != b.transposed,
                                   eights ? static_cast<const float *>(s->data_ptr()) : nullptr, (int)group, c.ptr, c.ld, (int)type, first != c.transposed, stream);
    }
    return result_of(st, args[4], std::move(C));
    END_HANDLE_TH_ERRORS
}

// A mixture-of-experts layer: what the C ABI gets of it, behind a capsule.  dtype -1: no part of it has a 16-bit type, the input's will do.
constexpr const char *kMoe = "b200spmm_moe_t";
struct Moe {
    b200spmm_moe_t m{};
    b200spmm_int4_t gate_up{}, down{};
    std::vector<Held> held;
};
void free_moe(PyObject *capsule) { delete static_cast<Moe *>(PyCapsule_GetPointer(capsule, kMoe)); }

// moe_layer(router or None, gate_up, down (capsules of Int4Matrix, or tensors), experts, hidden, inner, top_k, renormalize) -> capsule
PyObject *moe_layer(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 8) {
        PyErr_SetString(PyExc_TypeError, "moe_layer takes 8 arguments");
        return nullptr;
    }
    const int64_t E = PyLong_AsLongLong(args[3]), H = PyLong_AsLongLong(args[4]), I = PyLong_AsLongLong(args[5]), top = PyLong_AsLongLong(args[6]);
    if (PyErr_Occurred()) return nullptr;
    if (E < 1 || E > 1024) return refuse("there must be between 1 and 1024 experts");
    if (H < 1 || I < 1 || H > 0x1000000 || I > 0x1000000) return refuse("the hidden and inner sizes must lie between 1 and 2^24");
    if (top < 1 || top > 32) return refuse("top_k must lie between 1 and 32");
    if (args[0] != Py_None && top > E) return refuse("top_k must not be above the number of experts");
    auto layer = std::make_unique<Moe>();
    Moe &made = *layer;
    b200spmm_moe_t &m = made.m;
    m.experts = (uint64_t)E;
    m.hidden = (uint64_t)H;
    m.inner = (uint64_t)I;
    m.top_k = (int32_t)top;
    m.renormalize = args[7] == Py_True;
    m.dtype = m.device = -1;
    bool lost = false, one_type = true, one_device = true, cuda = true;
    auto joins = [&](const at::Tensor &t, bool typed) {
        const int type = type_code(t.scalar_type()), device = t.is_cuda() ? (int)t.get_device() : -2;
        cuda = cuda && t.is_cuda();
        one_type = one_type && (!typed || m.dtype == -1 || m.dtype == type);
        one_device = one_device && (m.device == -1 || m.device == device);
        if (typed) m.dtype = type;
        m.device = device;
        lost = lost || wants_gradient(t);
        made.held.emplace_back(t);
    };
    auto is_16 = [](const at::Tensor &t) { return (t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16) && t.layout() == at::kStrided && !t.is_neg(); };
    if (args[0] != Py_None) {
        const at::Tensor *r = THPVariable_Check(args[0]) ? &THPVariable_Unpack(args[0]) : nullptr;
        Rows at;
        if (!r || !is_16(*r) || r->dim() != 2 || r->size(0) != E || r->size(1) != H || !rows_of(*r, &at))
            return refuse("router must be a float16 or bfloat16 tensor [experts, hidden] with unit stride along its rows");
        joins(*r, true);
        m.router = at.ptr;
        m.ld_router = at.ld;
    }
    if (PyCapsule_IsValid(args[1], kInt4) != PyCapsule_IsValid(args[2], kInt4)) return refuse("gate_up and down must both be Int4Matrix, or both 16-bit tensors");
    if (PyCapsule_IsValid(args[1], kInt4)) {
        const auto *up = static_cast<const Int4 *>(PyCapsule_GetPointer(args[1], kInt4)), *down = static_cast<const Int4 *>(PyCapsule_GetPointer(args[2], kInt4));
        made.gate_up = up->m;
        made.down = down->m;
        for (const Int4 *codes : {up, down}) made.held.insert(made.held.end(), codes->held.begin(), codes->held.end());
        if (made.gate_up.rows != (uint64_t)(E * 2 * I) || made.gate_up.cols != (uint64_t)H || made.down.rows != (uint64_t)(E * H) || made.down.cols != (uint64_t)I)
            return refuse("gate_up must have experts x 2 inner rows of the hidden size, down experts x hidden rows of the inner size");
        one_device = one_device && made.gate_up.device == made.down.device && (m.device == -1 || m.device == made.gate_up.device);
        m.device = made.gate_up.device;
    } else {
        const int64_t rows[2] = {2 * I, H}, cols[2] = {H, I};
        for (int i = 0; i < 2; ++i) {
            const at::Tensor *w = THPVariable_Check(args[1 + i]) ? &THPVariable_Unpack(args[1 + i]) : nullptr;
            if (!w || !is_16(*w) || w->dim() != 3 || w->size(0) != E || w->size(1) != rows[i] || w->size(2) != cols[i])
                return refuse("gate_up must be [experts, 2 inner, hidden] and down [experts, hidden, inner], float16 or bfloat16");
            const int64_t ld = w->stride(1);
            if ((cols[i] > 1 && w->stride(2) != 1) || ld < cols[i] || ld % 8 != 0 || ld > 1 << 28 || (E > 1 && w->stride(0) != rows[i] * ld) || reinterpret_cast<uintptr_t>(w->data_ptr()) % 16 != 0)
                return refuse("rows of 16-bit experts must start on 16 bytes, a multiple of 8 elements apart, and experts follow one another: pad the last dimension");
            joins(*w, true);
            (i ? m.down_16 : m.gate_up_16) = w->data_ptr();
            (i ? m.ld_down : m.ld_gate_up) = ld;
        }
    }
    if (lost) return refuse(kNoGradient);
    if (!one_type) return refuse("the router and 16-bit experts must have one type");
    if (!cuda || !one_device) return refuse("all parts of the layer must be on one CUDA device");
    if (const char *fault = fault_of(made.held)) return refuse(fault);
    PyObject *out = PyCapsule_New(layer.get(), kMoe, free_moe);
    if (out) layer.release();
    return out;
    END_HANDLE_TH_ERRORS
}

// moe(capsule, X, out or None, routing wanted, ids or None, shares or None) -> (out, ids or None, shares or None), the first a status where it is a number
PyObject *moe(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
    HANDLE_TH_ERRORS
    if (n_args != 6) {
        PyErr_SetString(PyExc_TypeError, "moe takes 6 arguments");
        return nullptr;
    }
    const auto *layer = static_cast<const Moe *>(PyCapsule_GetPointer(args[0], kMoe));
    if (!layer) return nullptr;
    if (const char *fault = fault_of(layer->held)) return refuse(fault);
    b200spmm_moe_t m = layer->m;
    const at::Tensor *X = cuda_tensor(args[1]);
    Rows x, y;
    const bool typed = X && (X->scalar_type() == at::kHalf || X->scalar_type() == at::kBFloat16) && (m.dtype == -1 || type_code(X->scalar_type()) == m.dtype);
    if (!typed || X->dim() != 2 || X->size(1) != (int64_t)m.hidden || X->get_device() != m.device || !rows_of(*X, &x))
        return refuse("X must be a CUDA tensor [tokens, hidden] of the layer's 16-bit type, on its device, with unit stride along its rows");
    const int64_t tokens = X->size(0);
    if (tokens > 256) return refuse("a call takes up to 256 tokens");
    m.dtype = type_code(X->scalar_type());
    if (layer->gate_up.values || layer->gate_up.rows) {
        m.gate_up = &layer->gate_up;
        m.down = &layer->down;
    }
    const bool given = args[4] != Py_None, routing = args[3] == Py_True;
    if (!given && !m.router) return refuse("the layer has no router: give it the experts' ids and shares");
    bool lost = wants_gradient(*X);
    const at::Tensor *ids = nullptr, *shares = nullptr;
    if (given) {
        ids = cuda_tensor(args[4]);
        shares = cuda_tensor(args[5]);
        auto fits = [&](const at::Tensor *t) { return t && t->get_device() == m.device && t->dim() == 2 && t->size(0) == tokens && t->size(1) == m.top_k && t->is_contiguous(); };
        if (!fits(ids) || (ids->scalar_type() != at::kInt && ids->scalar_type() != at::kLong)) return refuse("ids must be a contiguous int32 or int64 tensor [tokens, top_k] on the layer's device");
        if (!fits(shares) || shares->scalar_type() != at::kFloat) return refuse("shares must be a contiguous float32 tensor [tokens, top_k] on the layer's device");
        lost = lost || wants_gradient(*shares);
    }
    at::Tensor Y, new_ids, new_shares, workspace;
    if (args[2] != Py_None) {
        const at::Tensor *t = cuda_tensor(args[2]);
        if (!t || t->scalar_type() != X->scalar_type() || t->get_device() != m.device || t->dim() != 2 || t->size(0) != tokens || t->size(1) != (int64_t)m.hidden || !rows_of(*t, &y))
            return refuse("out must be a tensor like X with unit stride along its rows");
        lost = lost || wants_gradient(*t);
    }
    if (lost) return refuse(kNoGradient);
    if (args[2] == Py_None) {
        Y = new_cuda({tokens, (int64_t)m.hidden}, X->scalar_type(), *X);
        y = {Y.data_ptr(), (int64_t)m.hidden};
    }
    if (routing) {
        new_ids = new_cuda({tokens, (int64_t)m.top_k}, at::kInt, *X);
        new_shares = new_cuda({tokens, (int64_t)m.top_k}, at::kFloat, *X);
    }
    uint64_t bytes = 0;
    int st = b200spmm_moe_workspace(&m, tokens, &bytes);
    if (st == B200SPMM_OK) {
        workspace = new_cuda({(int64_t)bytes}, at::kByte, *X);
        void *ws = workspace.data_ptr(), *stream = c10::cuda::getCurrentCUDAStream(X->get_device()).stream();
        int32_t *i = routing ? static_cast<int32_t *>(new_ids.data_ptr()) : nullptr;
        float *s = routing ? static_cast<float *>(new_shares.data_ptr()) : nullptr;
        const void *ids_in = given ? ids->data_ptr() : nullptr;
        const float *shares_in = given ? static_cast<const float *>(shares->data_ptr()) : nullptr;
        const int id_bytes = given && ids->scalar_type() == at::kLong ? 8 : 4;
        const ThreadsAllowed threads;
        st = given ? b200spmm_moe_experts(&m, x.ptr, x.ld, tokens, ids_in, id_bytes, shares_in, y.ptr, y.ld, ws, bytes, stream)
                   : b200spmm_moe(&m, x.ptr, x.ld, tokens, y.ptr, y.ld, i, s, ws, bytes, stream);
    }
    if (st != B200SPMM_OK) return three(PyLong_FromLong(st), again(Py_None), again(Py_None));
    written(args[2]);
    PyObject *a = Y.defined() ? THPVariable_Wrap(std::move(Y)) : again(args[2]);
    PyObject *b = routing ? THPVariable_Wrap(std::move(new_ids)) : again(Py_None), *c = routing ? THPVariable_Wrap(std::move(new_shares)) : again(Py_None);
    return three(a, b, c);
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
                         {"rms_norm", fast<rms_norm>(), METH_FASTCALL, nullptr},
                         {"int4_matrix", fast<int4_matrix>(), METH_FASTCALL, nullptr},
                         {"int4_product", fast<int4_product>(), METH_FASTCALL, nullptr},
                         {"moe_layer", fast<moe_layer>(), METH_FASTCALL, nullptr},
                         {"moe", fast<moe>(), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding(void) { return PyModule_Create(&module); }
