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
// (route_tokens of 64 tokens 12 us, linear of one token 18): route, sort, unsort and linear allocate their outputs and call the ABI, and record
// what autograd needs.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <optional>

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
//
// route, sort, unsort and linear answer None to a call for the general way.  What autograd has to record goes through nodes of its own
// below: a backward pass that enters the interpreter from the engine's thread costs some 50 us a node.

struct Entries {
    decltype(&nvfp4_last_error) last_error;
    decltype(&nvfp4_route_tokens) route;
    decltype(&nvfp4_route_tokens_backward) route_backward;
    decltype(&nvfp4_sort_tokens) sort;
    decltype(&nvfp4_unsort_tokens) unsort;
    decltype(&nvfp4_unsort_tokens_backward) unsort_backward;
    decltype(&nvfp4_linear) linear;
    decltype(&nvfp4_linear_dz_scaled) linear_dz;
    decltype(&nvfp4_linear_dx_scaled) linear_dx;
    decltype(&nvfp4_linear_dw_scaled) linear_dw;
} g_entry = {};

// bind_operators(addresses of the entries in the order of Entries)
PyObject* bind_operators(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    constexpr int kEntries = sizeof(Entries) / sizeof(void*);
    if (count != kEntries) { PyErr_SetString(PyExc_TypeError, "bind_operators() takes the addresses of the operators' entries"); return nullptr; }
    void* p[kEntries];
    for (int i = 0; i < kEntries; ++i) {
        p[i] = PyLong_AsVoidPtr(args[i]);
        if (p[i] == nullptr) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "a null address"); return nullptr; }
    }
    g_entry = Entries{reinterpret_cast<decltype(Entries::last_error)>(p[0]), reinterpret_cast<decltype(Entries::route)>(p[1]),
                      reinterpret_cast<decltype(Entries::route_backward)>(p[2]), reinterpret_cast<decltype(Entries::sort)>(p[3]),
                      reinterpret_cast<decltype(Entries::unsort)>(p[4]), reinterpret_cast<decltype(Entries::unsort_backward)>(p[5]),
                      reinterpret_cast<decltype(Entries::linear)>(p[6]), reinterpret_cast<decltype(Entries::linear_dz)>(p[7]),
                      reinterpret_cast<decltype(Entries::linear_dx)>(p[8]), reinterpret_cast<decltype(Entries::linear_dw)>(p[9])};
    Py_RETURN_NONE;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// NVFP4_DTYPE_* of a tensor's type, -1 for others
int dtype_code(at::ScalarType type)
{
    return type == at::kBFloat16 ? NVFP4_DTYPE_BF16 : type == at::kHalf ? NVFP4_DTYPE_F16 : type == at::kFloat ? NVFP4_DTYPE_F32 : -1;
}
// A tangent of forward mode: the general way refuses it.
bool has_tangent(const at::Tensor& t) { return t._fw_grad(0).defined(); }
// A 2-D tensor of one of the three types on the current device with contiguous rows that do not overlap, at least a row and a column.
const at::Tensor* matrix(PyObject* o)
{
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    return t.is_cuda() && t.layout() == at::kStrided && t.has_storage() && t.dim() == 2 && dtype_code(t.scalar_type()) >= 0 && t.size(0) >= 1 &&
                   t.size(1) >= 1 && t.size(0) <= INT32_MAX && t.size(1) <= INT32_MAX && (t.size(1) == 1 || t.stride(1) == 1) &&
                   (t.size(0) == 1 || t.stride(0) >= t.size(1)) && t.get_device() == c10::cuda::current_device() && !t.is_conj() && !t.is_neg() &&
                   !has_tangent(t)
               ? &t
               : nullptr;
}
// Row stride of such a tensor; of a single row its length
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
// A contiguous tensor of the given type beside `like`.
const at::Tensor* beside(PyObject* o, at::ScalarType type, int64_t dim, const at::Tensor& like)
{
    const at::Tensor* t = plain(o, type, dim);
    return t != nullptr && t->get_device() == like.get_device() && t->is_contiguous() && !t->is_neg() && !has_tangent(*t) ? t : nullptr;
}
bool wants_gradient(const at::Tensor* t) { return t != nullptr && t->requires_grad(); }
// A small int argument; false where it is none.
bool number(PyObject* o, int& value)
{
    const long v = PyLong_Check(o) ? PyLong_AsLong(o) : -1;
    if (PyErr_Occurred()) PyErr_Clear();
    value = static_cast<int>(v);
    return v >= 0 && v <= INT32_MAX;
}
// Results as the interpreter has them: a tensor, or a tuple of them
PyObject* wrapped(const variable_list& tensors)
{
    if (tensors.size() == 1) return THPVariable_Wrap(tensors[0]);
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
at::Tensor fresh(const at::Tensor& like, at::ScalarType type, at::IntArrayRef size) { return at::empty(size, like.options().dtype(type).requires_grad(false)); }
cudaStream_t stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
// An error of the library as an exception: in a forward call it sends the call the general way, which meets and names it again.
void check(int rc)
{
    TORCH_CHECK(rc == 0, "nvfp4_b200 error ", rc, ": ", g_entry.last_error());
}
template <typename F>
void forward(F&& launch)                 // holding the interpreter's lock
{
    int rc;
    {
        Unlocked unlocked;
        rc = launch();
    }
    check(rc);
}
template <typename T>
T* pointer(const at::Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
// The gradient of an output in rows that the kernels can read
at::Tensor in_rows(const at::Tensor& given)
{
    const at::Tensor t = given.is_neg() ? given.resolve_neg() : given;      // the memory holds the values with the other sign
    return t.size(0) > 0 && t.size(1) > 0 && t.stride(1) == 1 && t.stride(0) >= t.size(1) ? t : t.contiguous();
}
// Whether this backward pass asks for a gradient (autograd.grad names some; an argument may require one that it does not): `edge` counts the
// tensors among the node's arguments, of which missing ones are none.
bool wanted(AutogradContext* ctx, size_t edge, bool there = true) { return there && ctx->needs_input_grad(edge); }
// An argument of a node that may be missing: nodes take no undefined tensors
std::optional<at::Tensor> present(const at::Tensor& t) { return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt; }
// Gradients that were computed without being recorded: whoever differentiates them again gets an error instead of nothing.
variable_list once(variable_list grads)
{
    if (!at::GradMode::is_enabled()) return grads;
    for (at::Tensor& t : grads)
        if (t.defined()) t = t.detach().set_requires_grad(true);
    auto guard = std::make_shared<torch::autograd::DelayedError>("the gradients of this operator are computed once and cannot be differentiated again",
                                                                 static_cast<int64_t>(grads.size()));
    return (*guard)(std::move(grads));
}

variable_list route_forward(const at::Tensor& logits, int k, int scores, int renormalize)
{
    const int64_t tokens = logits.size(0);
    at::Tensor ids = fresh(logits, at::kLong, {tokens, k}), weights = fresh(logits, at::kFloat, {tokens, k});
    forward([&] {
        return g_entry.route(logits.data_ptr(), row_stride(logits), dtype_code(logits.scalar_type()), tokens, static_cast<int>(logits.size(1)), k, scores,
                             renormalize, pointer<int64_t>(ids), pointer<float>(weights), stream());
    });
    return {ids, weights};
}
struct RouteNode : torch::autograd::Function<RouteNode> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, int64_t k, int64_t scores, int64_t renormalize)
    {
        variable_list out = route_forward(logits, static_cast<int>(k), static_cast<int>(scores), static_cast<int>(renormalize));
        ctx->set_materialize_grads(false);
        ctx->mark_non_differentiable({out[0]});
        ctx->save_for_backward({logits, out[0]});
        ctx->saved_data["scores"] = scores;
        ctx->saved_data["renormalize"] = renormalize;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        if (!grads[1].defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &logits = saved[0], &ids = saved[1], g = grads[1].resolve_neg().contiguous();
        const c10::cuda::CUDAGuard guard(logits.device());
        at::Tensor dlogits = fresh(logits, logits.scalar_type(), logits.sizes());
        check(g_entry.route_backward(logits.data_ptr(), row_stride(logits), dtype_code(logits.scalar_type()), logits.size(0), static_cast<int>(logits.size(1)),
                                     static_cast<int>(ids.size(1)), static_cast<int>(ctx->saved_data["scores"].toInt()),
                                     static_cast<int>(ctx->saved_data["renormalize"].toInt()), pointer<int64_t>(ids), pointer<float>(g), dlogits.data_ptr(),
                                     stream()));
        return once({dlogits, at::Tensor(), at::Tensor(), at::Tensor()});
    }
};

// route(logits, k, scores code, renormalize) -> (ids, weights)
PyObject* route(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    int k, scores, renormalize;
    if (count != 4 || g_entry.route == nullptr || !number(args[1], k) || !number(args[2], scores) || !number(args[3], renormalize)) Py_RETURN_NONE;
    try {
        const at::Tensor* logits = matrix(args[0]);
        if (logits == nullptr || k < 1 || k > 32 || k > logits->size(1) || logits->size(1) > 1024) Py_RETURN_NONE;
        return wrapped(at::GradMode::is_enabled() && wants_gradient(logits) ? RouteNode::apply(*logits, k, scores, renormalize)
                                                                            : route_forward(*logits, k, scores, renormalize));
    } catch (const std::exception&) {
        Py_RETURN_NONE;
    }
}

variable_list sort_forward(const at::Tensor& x, const at::Tensor& ids, int experts, int alignment)
{
    const int64_t tokens = x.size(0), k = ids.size(1), hidden = x.size(1), n = tokens * k;
    const int64_t m = (n + std::min<int64_t>(experts, n) * (alignment - 1)) / alignment * alignment;
    at::Tensor rows = fresh(x, x.scalar_type(), {m, hidden}), place = fresh(x, at::kLong, {tokens, k}), source = fresh(x, at::kInt, {m}),
               m_indices = fresh(x, at::kInt, {m});
    forward([&] {
        return g_entry.sort(x.data_ptr(), row_stride(x), dtype_code(x.scalar_type()), tokens, static_cast<int>(k), static_cast<int>(hidden),
                            pointer<int64_t>(ids), experts, alignment, m, rows.data_ptr(), pointer<int64_t>(place), pointer<int32_t>(source),
                            pointer<int32_t>(m_indices), stream());
    });
    return {rows, place, source, m_indices};
}
at::Tensor sum_rows(const at::Tensor& rows, const at::Tensor& place, const at::Tensor& weights, bool locked)
{
    at::Tensor y = fresh(rows, rows.scalar_type(), {place.size(0), rows.size(1)});
    auto launch = [&] {
        return g_entry.unsort(rows.data_ptr(), row_stride(rows), dtype_code(rows.scalar_type()), rows.size(0), pointer<int64_t>(place),
                              pointer<float>(weights), place.size(0), static_cast<int>(place.size(1)), static_cast<int>(rows.size(1)), y.data_ptr(),
                              stream());
    };
    if (locked) forward(launch);
    else check(launch());
    return y;
}
struct SortNode : torch::autograd::Function<SortNode> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& ids, int64_t experts, int64_t alignment)
    {
        variable_list out = sort_forward(x, ids, static_cast<int>(experts), static_cast<int>(alignment));
        ctx->set_materialize_grads(false);
        ctx->mark_non_differentiable({out[1], out[2], out[3]});
        ctx->save_for_backward({out[1]});
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
        const c10::cuda::CUDAGuard guard(grads[0].device());
        return once({sum_rows(in_rows(grads[0]), ctx->get_saved_variables()[0], at::Tensor(), false), at::Tensor(), at::Tensor(), at::Tensor()});
    }
};

// sort(x, ids, num_experts, alignment) -> (rows, place, source, m_indices)
PyObject* sort(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    int experts, alignment;
    if (count != 4 || g_entry.sort == nullptr || !number(args[2], experts) || !number(args[3], alignment)) Py_RETURN_NONE;
    try {
        const at::Tensor* x = matrix(args[0]);
        const at::Tensor* ids = x == nullptr ? nullptr : beside(args[1], at::kLong, 2, *x);
        if (ids == nullptr || ids->size(0) != x->size(0) || ids->size(1) < 1 || experts < 1 || experts > 1024 || alignment < 1 || alignment > (1 << 20))
            Py_RETURN_NONE;
        const int64_t n = x->size(0) * std::min<int64_t>(ids->size(1), INT32_MAX);
        if (n > INT32_MAX || n + std::min<int64_t>(experts, n) * (alignment - 1) > INT32_MAX) Py_RETURN_NONE;
        return wrapped(at::GradMode::is_enabled() && wants_gradient(x) ? SortNode::apply(*x, *ids, experts, alignment)
                                                                       : sort_forward(*x, *ids, experts, alignment));
    } catch (const std::exception&) {
        Py_RETURN_NONE;
    }
}

struct UnsortNode : torch::autograd::Function<UnsortNode> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& rows, const std::optional<at::Tensor>& given, const at::Tensor& place,
                              const at::Tensor& source)
    {
        const at::Tensor weights = given.value_or(at::Tensor());
        const bool want_weights = weights.defined() && weights.requires_grad();
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({want_weights ? rows : at::Tensor(), weights, place, source});
        return sum_rows(rows, place, weights, true);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        variable_list out(4);
        if (!grads[0].defined()) return out;
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &rows = saved[0], &weights = saved[1], &place = saved[2], &source = saved[3], dy = in_rows(grads[0]);
        const c10::cuda::CUDAGuard guard(dy.device());
        const bool want_weights = wanted(ctx, 1, weights.defined());
        if (wanted(ctx, 0)) out[0] = fresh(dy, dy.scalar_type(), {source.size(0), dy.size(1)});
        if (want_weights) out[1] = fresh(dy, at::kFloat, place.sizes());
        check(g_entry.unsort_backward(dy.data_ptr(), row_stride(dy), want_weights ? rows.data_ptr() : nullptr, want_weights ? row_stride(rows) : dy.size(1),
                                      dtype_code(dy.scalar_type()), source.size(0), pointer<int64_t>(place), pointer<int32_t>(source),
                                      pointer<float>(weights), place.size(0), static_cast<int>(place.size(1)), static_cast<int>(dy.size(1)),
                                      pointer<void>(out[0]), pointer<float>(out[1]), stream()));
        return once(std::move(out));
    }
};

// unsort(rows, place, source, weights or None) -> y
PyObject* unsort(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    if (count != 4 || g_entry.unsort == nullptr) Py_RETURN_NONE;
    try {
        const at::Tensor* rows = matrix(args[0]);
        const at::Tensor* place = rows == nullptr ? nullptr : beside(args[1], at::kLong, 2, *rows);
        const at::Tensor* source = place == nullptr ? nullptr : beside(args[2], at::kInt, 1, *rows);
        if (source == nullptr || source->size(0) != rows->size(0) || place->size(0) < 1 || place->size(1) < 1 || place->size(1) > INT32_MAX) Py_RETURN_NONE;
        const at::Tensor* weights = nullptr;
        if (args[3] != Py_None) {
            weights = beside(args[3], at::kFloat, 2, *rows);
            if (weights == nullptr || weights->sizes() != place->sizes()) Py_RETURN_NONE;
        }
        const at::Tensor w = weights != nullptr ? *weights : at::Tensor();
        return THPVariable_Wrap(at::GradMode::is_enabled() && (wants_gradient(rows) || wants_gradient(weights)) ? UnsortNode::apply(*rows, present(w), *place, *source)
                                                                                                                : sum_rows(*rows, *place, w, true));
    } catch (const std::exception&) {
        Py_RETURN_NONE;
    }
}

// bias, residual and slopes may be undefined
at::Tensor linear_forward(const at::Tensor& x, const at::Tensor& w, const at::Tensor& bias, const at::Tensor& residual, int activation, bool out32,
                          const at::Tensor& slopes)
{
    const at::ScalarType out = out32 ? at::kFloat : x.scalar_type();
    const int64_t m = x.size(0), n = w.size(0);
    at::Tensor d = fresh(x, out, {m, n});
    forward([&] {
        return g_entry.linear(x.data_ptr(), row_stride(x), w.data_ptr(), row_stride(w), pointer<void>(bias), pointer<void>(residual),
                              residual.defined() ? row_stride(residual) : 0, d.data_ptr(), n, pointer<int16_t>(slopes), slopes.defined() ? slopes.size(1) : 0,
                              static_cast<int>(m), static_cast<int>(n), static_cast<int>(x.size(1)), dtype_code(x.scalar_type()), dtype_code(out),
                              activation, nullptr, stream());
    });
    return d;
}
struct LinearNode : torch::autograd::Function<LinearNode> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& given_bias,
                              const std::optional<at::Tensor>& given_residual, int64_t activation, bool out32)
    {
        const at::Tensor bias = given_bias.value_or(at::Tensor()), residual = given_residual.value_or(at::Tensor());
        const bool want_x = x.requires_grad(), want_w = w.requires_grad(), want_bias = bias.defined() && bias.requires_grad();
        at::Tensor slopes;
        if (activation != NVFP4_ACTIVATION_NONE && (want_x || want_w || want_bias)) slopes = fresh(x, at::kShort, {x.size(0), (w.size(0) + 7) / 8 * 8});
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({want_w ? x : at::Tensor(), want_x ? w : at::Tensor(), slopes});
        ctx->saved_data["bias"] = bias.defined();
        ctx->saved_data["residual"] = residual.defined();
        ctx->saved_data["type"] = static_cast<int64_t>(x.scalar_type());
        return linear_forward(x, w, bias, residual, static_cast<int>(activation), out32, slopes);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        variable_list out(6);
        if (!grads[0].defined()) return out;
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &w = saved[1], &slopes = saved[2];
        const bool has_bias = ctx->saved_data["bias"].toBool(), want_x = wanted(ctx, 0), want_w = wanted(ctx, 1), want_bias = wanted(ctx, 2, has_bias),
                   products = want_x || want_w;
        if (wanted(ctx, has_bias ? 3 : 2, ctx->saved_data["residual"].toBool())) out[3] = grads[0];
        if (products || want_bias) {
            const at::Tensor dd = in_rows(grads[0]);
            const c10::cuda::CUDAGuard guard(dd.device());
            const auto type = static_cast<at::ScalarType>(ctx->saved_data["type"].toInt());
            const int m = static_cast<int>(dd.size(0)), n = static_cast<int>(dd.size(1)), code = dtype_code(type);
            // without an activation the incoming gradient is dz itself, where it can be an operand
            const bool as_it_is = !slopes.defined() && dd.scalar_type() == type && row_stride(dd) % 8 == 0 && reinterpret_cast<uintptr_t>(dd.data_ptr()) % 16 == 0;
            at::Tensor dz = as_it_is ? dd : products ? fresh(dd, type, {m, (n + 7) / 8 * 8}) : at::Tensor();
            const int64_t ldz = dz.defined() ? row_stride(dz) : 0;
            // an FP32 gradient may lie outside of FP16
            const at::Tensor scale = products && type == at::kHalf && dd.scalar_type() == at::kFloat ? fresh(dd, at::kFloat, {1}) : at::Tensor();
            if (want_bias) out[2] = fresh(dd, type, {n});
            if (want_bias || (products && !as_it_is))
                check(g_entry.linear_dz(dd.data_ptr(), row_stride(dd), pointer<int16_t>(slopes), slopes.defined() ? slopes.size(1) : 0,
                                        as_it_is ? nullptr : pointer<void>(dz), ldz, pointer<void>(out[2]), m, n, code, dtype_code(dd.scalar_type()),
                                        pointer<float>(scale), stream()));
            if (want_x) {
                out[0] = fresh(dd, type, {m, w.size(1)});
                check(g_entry.linear_dx(dz.data_ptr(), ldz, w.data_ptr(), row_stride(w), out[0].data_ptr(), w.size(1), m, n, static_cast<int>(w.size(1)), code,
                                        pointer<float>(scale), nullptr, stream()));
            }
            if (want_w) {
                out[1] = fresh(dd, type, {n, x.size(1)});
                check(g_entry.linear_dw(dz.data_ptr(), ldz, x.data_ptr(), row_stride(x), out[1].data_ptr(), x.size(1), m, n, static_cast<int>(x.size(1)), code,
                                        pointer<float>(scale), nullptr, stream()));
            }
        }
        return once(std::move(out));
    }
};

// linear(x, w, bias or None, residual or None, activation code, FP32 output) -> d
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t count)
{
    int activation, out32;
    if (count != 6 || g_entry.linear == nullptr || !number(args[4], activation) || !number(args[5], out32)) Py_RETURN_NONE;
    try {
        const at::Tensor* x = matrix(args[0]);
        const at::Tensor* w = matrix(args[1]);
        if (x == nullptr || w == nullptr || x->scalar_type() == at::kFloat || w->scalar_type() != x->scalar_type() || w->size(1) != x->size(1)) Py_RETURN_NONE;
        at::Tensor bias, residual;
        if (args[2] != Py_None) {
            const at::Tensor* t = beside(args[2], x->scalar_type(), 1, *x);
            if (t == nullptr || t->size(0) != w->size(0)) Py_RETURN_NONE;
            bias = *t;
        }
        if (args[3] != Py_None) {
            const at::Tensor* t = matrix(args[3]);
            if (t == nullptr || t->scalar_type() != (out32 ? at::kFloat : x->scalar_type()) || t->size(0) != x->size(0) || t->size(1) != w->size(0))
                Py_RETURN_NONE;
            residual = *t;
        }
        const bool record = at::GradMode::is_enabled() && (wants_gradient(x) || wants_gradient(w) || (bias.defined() && bias.requires_grad()) ||
                                                           (residual.defined() && residual.requires_grad()));
        return THPVariable_Wrap(record ? LinearNode::apply(*x, *w, present(bias), present(residual), activation, out32 != 0)
                                       : linear_forward(*x, *w, bias, residual, activation, out32 != 0, at::Tensor()));
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
