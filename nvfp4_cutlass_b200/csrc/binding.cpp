// The grouped GEMM's call as a CPython function: reading six tensors' types, shapes and strides through the interpreter and
// converting twenty arguments for ctypes takes longer than a decode kernel runs (a decode call of 16 tokens,
// 32 of 256 experts, N = 1024, K = 2048: 11.5 us among others by the general way, 6.1 with this function, which then is the kernels'
// time, each overlapping the next).
//
// It takes ordinary calls only -- plain CUDA tensors of the current device, shapes and types that fit -- and answers None to
// anything else, tensors without storage included; _C.py then goes through its conditions one by one and names the one
// that does not hold.  The C ABI's entry point comes from the caller (bind), so that nothing here is linked to it.
//
// The same for the operators around it, which take a few microseconds on the GPU and took three to five times that in the interpreter
// (route_tokens of 64 tokens 12 us, linear of one token 18): route, sort, unsort and linear allocate their outputs and call the ABI; they
// leave calls that autograd has to record to Python, too.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>

#include "../../include/nvfp4_b200.h"

namespace {

decltype(&nvfp4_grouped_gemm_contiguous) g_gemm = nullptr;

// A torch.Tensor or Parameter whose memory is on a CUDA device, else nullptr.  dim < 0: any number of dimensions.
const at::Tensor* plain(PyObject* o, at::ScalarType type, int64_t dim)
{
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.layout() == at::kStrided && t.has_storage() && t.scalar_type() == type && (dim < 0 || t.dim() == dim) ? &t : nullptr;
}

// The interpreter goes on while the library launches, as it does under ctypes.
struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
};

PyObject* bind(PyObject*, PyObject* address)
{
    void* p = PyLong_AsVoidPtr(address);
    if (p == nullptr && PyErr_Occurred()) return nullptr;
    g_gemm = reinterpret_cast<decltype(g_gemm)>(p);
    Py_RETURN_NONE;
}

// contiguous(a, b, sfb, gw, d, m_indices, policy code, residual pass, orientation, m_alignment) -> error code, or None
PyObject* contiguous(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    if (count != 10) { PyErr_SetString(PyExc_TypeError, "contiguous() takes ten arguments"); return nullptr; }
    int option[4];
    for (int i = 0; i < 4; ++i) {
        const long value = PyLong_Check(args[6 + i]) ? PyLong_AsLong(args[6 + i]) : -1;
        if (PyErr_Occurred()) PyErr_Clear();
        if (value < 0 || value > INT32_MAX) Py_RETURN_NONE;
        option[i] = static_cast<int>(value);
    }
    try {
        const at::Tensor* a = plain(args[0], at::kBFloat16, 2);
        const at::Tensor* b = plain(args[1], at::kChar, 2);
        const at::Tensor* sfb = plain(args[2], at::kInt, 2);
        const at::Tensor* gw = plain(args[3], at::kFloat, -1);
        const at::Tensor* d = plain(args[4], at::kBFloat16, 2);
        const at::Tensor* m_indices = plain(args[5], at::kInt, 1);
        if (g_gemm == nullptr || a == nullptr || b == nullptr || sfb == nullptr || gw == nullptr || d == nullptr || m_indices == nullptr)
            Py_RETURN_NONE;
        const int64_t m = a->size(0), k = a->size(1), n = d->size(1), e = gw->numel();
        if (m > INT32_MAX || k > INT32_MAX || n > INT32_MAX || e > INT32_MAX || d->size(0) != m || m_indices->size(0) != m || b->size(0) != e * n ||
            b->size(1) != k / 2 || sfb->size(0) != e * (k / 64) || sfb->size(1) != n || a->stride(1) != 1 || d->stride(1) != 1 ||
            !b->is_contiguous() || !sfb->is_contiguous() || !gw->is_contiguous() || !m_indices->is_contiguous())
            Py_RETURN_NONE;
        const auto device = a->get_device();
        if (b->get_device() != device || sfb->get_device() != device || gw->get_device() != device || d->get_device() != device ||
            m_indices->get_device() != device || c10::cuda::current_device() != device)
            Py_RETURN_NONE;
        // the stride of a single row is not used, and may be anything
        const int64_t lda = m > 1 ? a->stride(0) : std::max<int64_t>(a->stride(0), k), ldd = m > 1 ? d->stride(0) : std::max<int64_t>(d->stride(0), n);
        const void *pa = a->data_ptr(), *pb = b->data_ptr(), *psfb = sfb->data_ptr(), *pm = m_indices->data_ptr();
        const float* pgw = static_cast<const float*>(gw->data_ptr());
        void* pd = d->data_ptr();
        cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
        int rc = 0;
        {
            Unlocked unlocked;
            rc = g_gemm(pa, lda, pb, psfb, pgw, pd, ldd, static_cast<const int32_t*>(pm), static_cast<int>(m), static_cast<int>(n),
                        static_cast<int>(k), static_cast<int>(e), option[0], option[1], option[2], option[3], nullptr, nullptr, stream);
        }
        return PyLong_FromLong(rc);
    } catch (const std::exception&) {       // a tensor that has no memory to point at: the general path says so
        Py_RETURN_NONE;
    }
}

// ---- operators around the GEMM -----------------------------------------------------------------------------------

decltype(&nvfp4_route_tokens) g_route = nullptr;
decltype(&nvfp4_sort_tokens) g_sort = nullptr;
decltype(&nvfp4_unsort_tokens) g_unsort = nullptr;
decltype(&nvfp4_linear) g_linear = nullptr;

// bind_operators(addresses of nvfp4_route_tokens, nvfp4_sort_tokens, nvfp4_unsort_tokens, nvfp4_linear)
PyObject* bind_operators(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    if (count != 4) { PyErr_SetString(PyExc_TypeError, "bind_operators() takes four addresses"); return nullptr; }
    void* p[4];
    for (int i = 0; i < 4; ++i) {
        p[i] = PyLong_AsVoidPtr(args[i]);
        if (p[i] == nullptr && PyErr_Occurred()) return nullptr;
    }
    g_route = reinterpret_cast<decltype(g_route)>(p[0]);
    g_sort = reinterpret_cast<decltype(g_sort)>(p[1]);
    g_unsort = reinterpret_cast<decltype(g_unsort)>(p[2]);
    g_linear = reinterpret_cast<decltype(g_linear)>(p[3]);
    Py_RETURN_NONE;
}

// NVFP4_DTYPE_* of a tensor's type, -1 for others
int dtype_code(at::ScalarType type)
{
    return type == at::kBFloat16 ? NVFP4_DTYPE_BF16 : type == at::kHalf ? NVFP4_DTYPE_F16 : type == at::kFloat ? NVFP4_DTYPE_F32 : -1;
}
// A 2-D tensor of one of the three types on the current device with contiguous rows that do not overlap, at least a row and a column, that
// needs no gradient; ld: its row stride (of a single row: its length).
const at::Tensor* matrix(PyObject* o, int64_t& ld)
{
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() || t.dim() != 2 || dtype_code(t.scalar_type()) < 0 || t.size(0) < 1 || t.size(1) < 1 ||
        t.size(0) > INT32_MAX || t.size(1) > INT32_MAX || (t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1)) ||
        t.get_device() != c10::cuda::current_device() || t.is_conj() || t.is_neg() || (t.requires_grad() && at::GradMode::is_enabled()))
        return nullptr;
    ld = t.size(0) > 1 ? t.stride(0) : t.size(1);
    return &t;
}
// A contiguous tensor of the given type beside `like` that needs no gradient.
const at::Tensor* beside(PyObject* o, at::ScalarType type, int64_t dim, const at::Tensor& like)
{
    const at::Tensor* t = plain(o, type, dim);
    return t != nullptr && t->get_device() == like.get_device() && t->is_contiguous() && !(t->requires_grad() && at::GradMode::is_enabled()) ? t : nullptr;
}
// A small int argument; false where it is none.
bool number(PyObject* o, int& value)
{
    const long v = PyLong_Check(o) ? PyLong_AsLong(o) : -1;
    if (PyErr_Occurred()) PyErr_Clear();
    value = static_cast<int>(v);
    return v >= 0 && v <= INT32_MAX;
}
// Results as the interpreter has them: a tensor, or a tuple of them
PyObject* wrapped(std::initializer_list<at::Tensor> tensors)
{
    if (tensors.size() == 1) return THPVariable_Wrap(*tensors.begin());
    PyObject* tuple = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
    if (tuple == nullptr) return nullptr;
    Py_ssize_t i = 0;
    for (const at::Tensor& t : tensors) {
        PyObject* o = THPVariable_Wrap(t);
        if (o == nullptr) { Py_DECREF(tuple); return nullptr; }
        PyTuple_SET_ITEM(tuple, i++, o);
    }
    return tuple;
}
template <typename F>
int unlocked(F&& launch)
{
    Unlocked state;
    return launch();
}
at::Tensor fresh(const at::Tensor& like, at::ScalarType type, at::IntArrayRef size) { return at::empty(size, like.options().dtype(type).requires_grad(false)); }

// The four below answer an error code of the library, or None to a call for the general way.

// route(logits, k, scores code, renormalize) -> (ids, weights)
PyObject* route(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    int64_t ld;
    int k, scores, renormalize;
    if (count != 4 || g_route == nullptr || !number(args[1], k) || !number(args[2], scores) || !number(args[3], renormalize)) Py_RETURN_NONE;
    try {
        const at::Tensor* logits = matrix(args[0], ld);
        if (logits == nullptr || k < 1 || k > 32 || k > logits->size(1) || logits->size(1) > 1024) Py_RETURN_NONE;
        const int64_t tokens = logits->size(0);
        at::Tensor ids = fresh(*logits, at::kLong, {tokens, k}), weights = fresh(*logits, at::kFloat, {tokens, k});
        const int rc = unlocked([&] { return g_route(logits->data_ptr(), ld, dtype_code(logits->scalar_type()), tokens, static_cast<int>(logits->size(1)), k, scores, renormalize,
                               ids.data_ptr<int64_t>(), weights.data_ptr<float>(), c10::cuda::getCurrentCUDAStream().stream()); });
        return rc == 0 ? wrapped({ids, weights}) : PyLong_FromLong(rc);
    } catch (const std::exception&) {
        Py_RETURN_NONE;
    }
}

// sort(x, ids, num_experts, alignment) -> (rows, place, source, m_indices)
PyObject* sort(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    int64_t ld;
    int experts, alignment;
    if (count != 4 || g_sort == nullptr || !number(args[2], experts) || !number(args[3], alignment)) Py_RETURN_NONE;
    try {
        const at::Tensor* x = matrix(args[0], ld);
        const at::Tensor* ids = x == nullptr ? nullptr : beside(args[1], at::kLong, 2, *x);
        if (ids == nullptr || ids->size(0) != x->size(0) || ids->size(1) < 1 || experts < 1 || experts > 1024 || alignment < 1 || alignment > (1 << 20))
            Py_RETURN_NONE;
        const int64_t tokens = x->size(0), k = ids->size(1), hidden = x->size(1);
        if (k > INT32_MAX / tokens) Py_RETURN_NONE;
        const int64_t n = tokens * k, m = (n + std::min<int64_t>(experts, n) * (alignment - 1)) / alignment * alignment;
        if (m > INT32_MAX) Py_RETURN_NONE;
        at::Tensor rows = fresh(*x, x->scalar_type(), {m, hidden}), place = fresh(*x, at::kLong, {tokens, k}), source = fresh(*x, at::kInt, {m}),
                   m_indices = fresh(*x, at::kInt, {m});
        const int rc = unlocked([&] { return g_sort(x->data_ptr(), ld, dtype_code(x->scalar_type()), tokens, static_cast<int>(k), static_cast<int>(hidden), ids->data_ptr<int64_t>(),
                              experts, alignment, m, rows.data_ptr(), place.data_ptr<int64_t>(), source.data_ptr<int32_t>(), m_indices.data_ptr<int32_t>(),
                              c10::cuda::getCurrentCUDAStream().stream()); });
        return rc == 0 ? wrapped({rows, place, source, m_indices}) : PyLong_FromLong(rc);
    } catch (const std::exception&) {
        Py_RETURN_NONE;
    }
}

// unsort(rows, place, weights or None) -> y
PyObject* unsort(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    int64_t ld;
    if (count != 3 || g_unsort == nullptr) Py_RETURN_NONE;
    try {
        const at::Tensor* rows = matrix(args[0], ld);
        const at::Tensor* place = rows == nullptr ? nullptr : beside(args[1], at::kLong, 2, *rows);
        if (place == nullptr || place->size(0) < 1 || place->size(1) < 1 || place->size(1) > INT32_MAX) Py_RETURN_NONE;
        const at::Tensor* weights = nullptr;
        if (args[2] != Py_None) {
            weights = beside(args[2], at::kFloat, 2, *rows);
            if (weights == nullptr || weights->sizes() != place->sizes()) Py_RETURN_NONE;
        }
        const int64_t tokens = place->size(0), hidden = rows->size(1);
        at::Tensor y = fresh(*rows, rows->scalar_type(), {tokens, hidden});
        const int rc = unlocked([&] { return g_unsort(rows->data_ptr(), ld, dtype_code(rows->scalar_type()), rows->size(0), place->data_ptr<int64_t>(),
                                weights != nullptr ? weights->data_ptr<float>() : nullptr, tokens, static_cast<int>(place->size(1)),
                                static_cast<int>(hidden), y.data_ptr(), c10::cuda::getCurrentCUDAStream().stream()); });
        return rc == 0 ? wrapped({y}) : PyLong_FromLong(rc);
    } catch (const std::exception&) {
        Py_RETURN_NONE;
    }
}

// linear(x, w, bias or None, residual or None, activation code, FP32 output) -> d
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    int64_t ldx, ldw, ldr = 0;
    int activation, out32;
    if (count != 6 || g_linear == nullptr || !number(args[4], activation) || !number(args[5], out32)) Py_RETURN_NONE;
    try {
        const at::Tensor* x = matrix(args[0], ldx);
        const at::Tensor* w = matrix(args[1], ldw);
        if (x == nullptr || w == nullptr || x->scalar_type() == at::kFloat || w->scalar_type() != x->scalar_type() || w->size(1) != x->size(1)) Py_RETURN_NONE;
        const int64_t m = x->size(0), n = w->size(0), k = x->size(1);
        const at::ScalarType out = out32 ? at::kFloat : x->scalar_type();
        const at::Tensor *bias = nullptr, *residual = nullptr;
        if (args[2] != Py_None) {
            bias = beside(args[2], x->scalar_type(), 1, *x);
            if (bias == nullptr || bias->size(0) != n) Py_RETURN_NONE;
        }
        if (args[3] != Py_None) {
            residual = matrix(args[3], ldr);
            if (residual == nullptr || residual->scalar_type() != out || residual->size(0) != m || residual->size(1) != n) Py_RETURN_NONE;
        }
        at::Tensor d = fresh(*x, out, {m, n});
        const int rc = unlocked([&] { return g_linear(x->data_ptr(), ldx, w->data_ptr(), ldw, bias != nullptr ? bias->data_ptr() : nullptr,
                                residual != nullptr ? residual->data_ptr() : nullptr, ldr, d.data_ptr(), n, nullptr, 0, static_cast<int>(m),
                                static_cast<int>(n), static_cast<int>(k), dtype_code(x->scalar_type()), dtype_code(out), activation, nullptr,
                                c10::cuda::getCurrentCUDAStream().stream()); });
        return rc == 0 ? wrapped({d}) : PyLong_FromLong(rc);
    } catch (const std::exception&) {
        Py_RETURN_NONE;
    }
}

PyMethodDef kMethods[] = {
    {"bind", bind, METH_O, nullptr},
    {"contiguous", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(contiguous)), METH_FASTCALL, nullptr},
    {"bind_operators", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind_operators)), METH_FASTCALL, nullptr},
    {"route", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(route)), METH_FASTCALL, nullptr},
    {"sort", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(sort)), METH_FASTCALL, nullptr},
    {"unsort", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(unsort)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&kModule); }
