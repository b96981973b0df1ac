// Python binding of the operators whose small calls are bound by the host: checks of arguments, allocation of outputs and the call of
// the C ABI (include/coat_hip.h) in one compiled step.  The kernels stay behind the C ABI; this module is handed the library's entry
// points at load time (bind) and launches nothing itself.
//
// Measured against the same steps in Python over ctypes: a LayerNorm forward of [4, 4096] 12 us a call there, a step of 192 tensors
// 336 us (1.7 us a tensor for five attribute calls on each of five lists).
//
// Errors: ValueError and RuntimeError as the rest of the package raises them; nothing is launched before everything is checked.
#include <Python.h>

#include <ATen/TracerMode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "../../include/coat_hip.h"

namespace {

#define ENTRY_POINTS(X)          \
    X(coat_status_string)        \
    X(coat_layer_norm_forward)   \
    X(coat_layer_norm_partials)  \
    X(coat_layer_norm_backward)  \
    X(coat_rope_axes)            \
    X(coat_grad_norm_partials)   \
    X(coat_grad_norm_multi)      \
    X(coat_adamw_step_multi)
struct {
#define POINTER(name) decltype(&::name) name;
    ENTRY_POINTS(POINTER)
#undef POINTER
} lib;
PyObject* raw_stream = nullptr;  // device index -> handle of torch's current stream

// ------------------------------------------------------------------------------------------------ arguments
const at::Tensor* tensor_or_none(PyObject* o, const char* who, const char* name) {
    if (o == Py_None) return nullptr;
    TORCH_CHECK_TYPE(THPVariable_Check(o), who, ": ", name, " must be a tensor");
    return &THPVariable_Unpack(o);
}
const at::Tensor& tensor(PyObject* o, const char* who, const char* name) {
    const at::Tensor* t = tensor_or_none(o, who, name);
    TORCH_CHECK_TYPE(t, who, ": ", name, " must be a tensor");
    return *t;
}
bool truth(PyObject* o) {
    const int t = PyObject_IsTrue(o);
    if (t < 0) throw python_error();
    return t != 0;
}
double real(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
int64_t whole(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
void arguments(const char* who, Py_ssize_t got, Py_ssize_t wanted) {
    TORCH_CHECK_TYPE(got == wanted, who, ": ", wanted, " arguments are needed, got ", got);
    TORCH_CHECK(raw_stream, who, ": the binding has no library yet");
}

// torch does not see what is computed here: a forward-mode tangent would be lost and read as a zero derivative, a recorded program would
// return memory that nothing fills.  Both are refused.  Inside an autograd function, where torch turns forward mode off, they are that
// function's concern (it refuses tangents itself and is recorded as one step), but for a recording of dispatched operations, which
// goes through it.
bool forward_mode() {
    return c10::AutogradState::get_tls_state().get_fw_grad_mode() && torch::autograd::ForwardADLevel::try_get_by_idx(0);
}
void no_tangent(const at::Tensor& t, const char* who) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), who, ": forward-mode derivatives are not implemented");
}
void unrecorded(const char* who, std::initializer_list<const at::Tensor*> tensors) {
    const bool recorded = c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value() ||
                          (at::tracer::impl::is_dispatch_enabled() && c10::AutogradState::get_tls_state().get_fw_grad_mode());
    TORCH_CHECK_NOT_IMPLEMENTED(!recorded, who, ": a trace cannot record this call");
    if (forward_mode())
        for (const at::Tensor* t : tensors)
            if (t) no_tangent(*t, who);
}

const char* name_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return "torch.float32";
        case at::kBFloat16: return "torch.bfloat16";
        case at::kHalf: return "torch.float16";
        case at::kDouble: return "torch.float64";
        default: return c10::toString(t);
    }
}
int code_of(at::ScalarType t) {
    if (t == at::kFloat) return COAT_F32;
    if (t == at::kBFloat16) return COAT_BF16;
    TORCH_CHECK_VALUE(t == at::kHalf, "unsupported dtype ", name_of(t));
    return COAT_F16;
}
void on_gpu(const at::Tensor& t) {
    TORCH_CHECK(t.is_cuda(), "coat_amd kernels need tensors on the GPU (got a ", c10::DeviceTypeName(t.device().type(), true), " tensor)");
}
void* stream_of(const at::Tensor& t) {
    PyObject* index = PyLong_FromLong(t.get_device());
    if (!index) throw python_error();
    PyObject* handle = PyObject_CallFunctionObjArgs(raw_stream, index, nullptr);
    Py_DECREF(index);
    if (!handle) throw python_error();
    void* s = PyLong_AsVoidPtr(handle);
    Py_DECREF(handle);
    if (!s && PyErr_Occurred()) throw python_error();
    return s;
}
void check(int status, const char* who) {
    if (status == COAT_OK) return;
    const char* what = lib.coat_status_string(status);
    TORCH_CHECK_VALUE(status != COAT_EINVAL && status != COAT_ESHAPE && status != COAT_EDTYPE && status != COAT_EALIGN, who, ": ", what);
    TORCH_CHECK(false, who, ": ", what);
}
at::Tensor dense_like(const at::Tensor& t) { return t.is_contiguous() ? at::empty_like(t) : at::empty(t.sizes(), t.options()); }
void* data(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

PyObject* tuple(std::initializer_list<at::Tensor> tensors) {
    PyObject* out = PyTuple_New((Py_ssize_t)tensors.size());
    if (!out) throw python_error();
    Py_ssize_t i = 0;
    for (const at::Tensor& t : tensors) {
        PyObject* o = t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None);
        if (!o) {
            Py_DECREF(out);
            throw python_error();
        }
        PyTuple_SET_ITEM(out, i++, o);
    }
    return out;
}

// ------------------------------------------------------------------------------------------------ LayerNorm
// The rows of t at one distance (in elements): t itself wherever they lie so, else a copy.
at::Tensor rows(const at::Tensor& t, int64_t N, int64_t& pitch) {
    pitch = N;
    if (t.is_contiguous() || t.numel() == 0) return t;
    bool even = N == 1 || t.stride(-1) == 1;
    int64_t first = -1, expected = -1;
    for (int64_t d = t.dim() - 2; d >= 0 && even; d--) {
        if (t.size(d) == 1) continue;
        if (first < 0) first = t.stride(d);
        else even = t.stride(d) == expected;
        expected = t.stride(d) * t.size(d);
    }
    if (!even || (first >= 0 && first < N)) return t.contiguous();  // also rows that overlap, or one row repeated
    if (first >= 0) pitch = first;
    return t;
}

void norm_arguments(const char* who, const at::Tensor& x, const at::Tensor* w, const at::Tensor* b) {
    on_gpu(x);
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, who, ": expected a tensor with a last dimension to normalise over, got shape ", x.sizes());
    code_of(x.scalar_type());
    TORCH_CHECK_VALUE(w || !b, who, ": a bias needs a weight");
    for (const at::Tensor* p : {w, b}) {
        if (!p) continue;
        const char* name = p == w ? "weight" : "bias";
        TORCH_CHECK_VALUE(p->dim() == 1 && p->size(0) == x.size(-1), who, ": ", name, " must have shape [", x.size(-1), "], got ", p->sizes());
        TORCH_CHECK_VALUE(p->device() == x.device(), who, ": ", name, " is on ", p->device(), ", x on ", x.device());
        code_of(p->scalar_type());
    }
    TORCH_CHECK_VALUE(!b || b->scalar_type() == w->scalar_type(), who, ": bias dtype differs from weight dtype");
}

// (x, weight, bias, eps) -> (y, mean, rstd)
PyObject* layer_norm_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const char* who = "layer_norm_forward";
    arguments(who, n, 4);
    const at::Tensor& x = tensor(a[0], who, "x");
    const at::Tensor *w = tensor_or_none(a[1], who, "weight"), *b = tensor_or_none(a[2], who, "bias");
    const double eps = real(a[3]);
    unrecorded(who, {&x, w, b});
    norm_arguments(who, x, w, b);
    TORCH_CHECK_VALUE(eps >= 0.0, who, ": invalid eps ", eps);
    const c10::DeviceGuard guard(x.device());
    const int64_t N = x.size(-1);
    at::Tensor y = dense_like(x), mean = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat)), rstd = at::empty_like(mean);
    int64_t pitch;
    const at::Tensor xr = rows(x, N, pitch);
    const at::Tensor wc = w ? w->contiguous() : at::Tensor(), bc = b ? b->contiguous() : at::Tensor();
    check(lib.coat_layer_norm_forward(xr.data_ptr(), pitch, code_of(x.scalar_type()), data(wc), data(bc), w ? code_of(w->scalar_type()) : 0,
                                      y.data_ptr(), (float*)mean.data_ptr(), (float*)rstd.data_ptr(), x.numel() / N, N, (float)eps, stream_of(x)),
          who);
    return tuple({y, mean, rstd});
    END_HANDLE_TH_ERRORS
}

// (dy, x, mean, rstd, weight, x_grad, weight_grad, bias_grad) -> (dx, dw, db)
PyObject* layer_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const char* who = "layer_norm_backward";
    arguments(who, n, 8);
    const at::Tensor &dy = tensor(a[0], who, "dy"), &x = tensor(a[1], who, "x"), &mean = tensor(a[2], who, "mean"), &rstd = tensor(a[3], who, "rstd");
    const at::Tensor* w = tensor_or_none(a[4], who, "weight");
    unrecorded(who, {&dy, &x, &mean, &rstd, w});
    norm_arguments(who, x, w, nullptr);
    const int64_t N = x.size(-1), M = x.numel() / N;
    TORCH_CHECK_VALUE(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && dy.device() == x.device(), who,
                      ": dy must have x's shape, dtype and device");
    for (const at::Tensor* t : {&mean, &rstd})
        TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->numel() == M && t->device() == x.device() && t->is_contiguous(), who, ": ",
                          t == &mean ? "mean" : "rstd", " must be contiguous fp32 with one element a row, on x's device");
    const c10::DeviceGuard guard(x.device());
    const at::Tensor wc = w ? w->contiguous() : at::Tensor();
    at::Tensor dx, dw, db, partial;
    if (truth(a[5])) dx = dense_like(x);
    if (w && truth(a[6])) dw = at::empty_like(wc);
    if (w && truth(a[7])) db = at::empty_like(wc);
    const int64_t wanted = dw.defined() + db.defined();
    int parts = 0;
    if (wanted) {
        parts = lib.coat_layer_norm_partials(M, N);
        if (parts < 0) check(parts, who);
        if (parts > 1 || N > COAT_LAYER_NORM_ROW) partial = at::empty({wanted, parts, N}, x.options().dtype(at::kFloat));  // one block needs none
    }
    int64_t x_pitch, dy_pitch;
    const at::Tensor xr = rows(x, N, x_pitch), gr = rows(dy, N, dy_pitch);
    check(lib.coat_layer_norm_backward(gr.data_ptr(), dy_pitch, xr.data_ptr(), x_pitch, code_of(x.scalar_type()), (const float*)mean.data_ptr(),
                                       (const float*)rstd.data_ptr(), data(wc), w ? code_of(w->scalar_type()) : 0, data(dx), data(dw), data(db),
                                       (float*)data(partial), parts, M, N, stream_of(x)),
          who);
    return tuple({dx, dw, db});
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------------ rotary
// (q, k, positions, turns, axis, head_dim, axes, pairs, adjacent, inverse, stream of the tables) -> (q, k)
PyObject* rotary_axes(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const char* who = "rotary_axes";
    arguments(who, n, 11);
    const at::Tensor *q = tensor_or_none(a[0], who, "q"), *k = tensor_or_none(a[1], who, "k");
    at::Tensor pos = tensor(a[2], who, "position_ids");
    const at::Tensor &turns = tensor(a[3], who, "turns"), &axis = tensor(a[4], who, "axis");
    const int64_t D = whole(a[5]), axes = whole(a[6]), pairs = whole(a[7]);
    TORCH_CHECK_VALUE(q || k, who, ": neither q nor k given");
    unrecorded(who, {q, k});
    TORCH_CHECK_VALUE(turns.scalar_type() == at::kDouble && turns.numel() == pairs && turns.is_contiguous() && axis.scalar_type() == at::kInt &&
                          axis.numel() == pairs && axis.is_contiguous(),
                      who, ": the plan's tables must be contiguous, fp64 and int32, with one element for each of ", pairs, " pairs");
    const at::Tensor& first = q ? *q : *k;
    on_gpu(first);
    for (const at::Tensor* t : {q, k}) {
        if (!t) continue;
        TORCH_CHECK_VALUE(t->dim() == 4 && first.dim() == 4 && t->size(0) == first.size(0) && t->size(1) == first.size(1) && t->size(3) == D, who,
                          ": expected [batch, seq, heads, ", D, "] tensors of one batch, got ", t->sizes());
        TORCH_CHECK_VALUE(t->scalar_type() == first.scalar_type() && t->device() == first.device(), who, ": q and k must have one dtype and device");
    }
    TORCH_CHECK_VALUE(turns.device() == first.device() && axis.device() == first.device(), who, ": the plan's tables are on ", turns.device(),
                      " and ", axis.device(), ", q and k on ", first.device());
    const int dt = code_of(first.scalar_type());
    const int64_t B = first.size(0), S = first.size(1);
    TORCH_CHECK_VALUE(pos.dim() == 3 && pos.size(0) == axes, who, ": expected position_ids of shape [", axes, ", batch, seq], got ", pos.sizes());
    TORCH_CHECK_VALUE(pos.device() == first.device(), who, ": position_ids are on ", pos.device(), ", q and k on ", first.device());
    TORCH_CHECK_VALUE(at::isIntegralType(pos.scalar_type(), false), who, ": position_ids must be whole numbers, got ", name_of(pos.scalar_type()));
    const c10::DeviceGuard guard(first.device());
    if (pos.scalar_type() != at::kLong) pos = pos.to(at::kLong);
    if (pos.size(1) != B || pos.size(2) != S) pos = pos.expand({axes, B, S});
    void *const stream = stream_of(first), *const home = PyLong_AsVoidPtr(a[10]);
    if (!home && PyErr_Occurred()) throw python_error();
    at::Tensor in[2], out[2];
    int64_t strides[2][3] = {};
    int heads[2] = {};
    for (int i = 0; i < 2; i++) {
        const at::Tensor* t = i == 0 ? q : k;
        if (!t) continue;
        TORCH_CHECK_VALUE(t->size(2) <= 1024, who, ": at most 1024 heads");
        in[i] = t->stride(3) == 1 ? *t : t->contiguous();
        out[i] = dense_like(in[i]);
        heads[i] = (int)t->size(2);
        for (int d = 0; d < 3; d++) strides[i][d] = in[i].stride(d);
    }
    check(lib.coat_rope_axes(data(in[0]), data(out[0]), strides[0][0], strides[0][1], strides[0][2], heads[0], data(in[1]), data(out[1]),
                             strides[1][0], strides[1][1], strides[1][2], heads[1], dt, (const int64_t*)pos.data_ptr(), pos.stride(0),
                             pos.stride(1), pos.stride(2), (int)axes, (const double*)turns.data_ptr(), (const int32_t*)axis.data_ptr(), (int)pairs,
                             (int)D, truth(a[8]), truth(a[9]), B, S, stream),
          who);
    if (stream != home) {  // the caller cannot see the tables: kept from reuse until this stream has read them, should their plan be dropped
        const c10::Stream current = c10::impl::VirtualGuardImpl(first.device().type()).getStream(first.device());
        turns.record_stream(current);
        axis.record_stream(current);
    }
    return tuple({out[0], out[1]});
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------------ lists of tensors
// A list or tuple of tensors, kept alive while it is used.
struct List {
    PyObject* fast;
    List(PyObject* o, const char* who, const char* name) : fast(PySequence_Fast(o, "")) {
        if (!fast) {
            PyErr_Clear();
            TORCH_CHECK_TYPE(false, who, ": ", name, " must be a list of tensors");
        }
        for (Py_ssize_t i = 0; i < size(); i++)
            if (!THPVariable_Check(PySequence_Fast_GET_ITEM(fast, i))) {
                Py_DECREF(fast);
                TORCH_CHECK_TYPE(false, who, ": ", name, " must be a list of tensors");
            }
    }
    List(const List&) = delete;
    ~List() { Py_DECREF(fast); }
    Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(fast); }
    const at::Tensor& operator[](Py_ssize_t i) const { return THPVariable_Unpack(PySequence_Fast_GET_ITEM(fast, i)); }
};

// (grads, max_norm) -> fp32 [2]: norm, factor.  grads is not empty.
PyObject* grad_norm_multi(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const char* who = "grad_norm_multi";
    arguments(who, n, 2);
    const List grads(a[0], who, "grads");
    const double max_norm = real(a[1]);
    const Py_ssize_t count = grads.size();
    TORCH_CHECK_VALUE(count > 0, who, ": no gradients");
    unrecorded(who, {});
    if (forward_mode())
        for (Py_ssize_t i = 0; i < count; i++) no_tangent(grads[i], who);
    const at::Device device = grads[0].device();
    on_gpu(grads[0]);
    const c10::DeviceGuard guard(device);
    std::vector<at::Tensor> copies;
    std::vector<const void*> address(count);
    std::vector<int> kind(count);
    std::vector<int64_t> numel(count);
    for (Py_ssize_t i = 0; i < count; i++) {
        const at::Tensor& g = grads[i];
        TORCH_CHECK(g.device() == device, who, ": grads holds tensors that are not on the first tensor's device");
        kind[i] = code_of(g.scalar_type());
        numel[i] = g.numel();
        if (g.is_contiguous()) {
            address[i] = g.data_ptr();
        } else {
            copies.push_back(g.contiguous());
            address[i] = copies.back().data_ptr();
        }
    }
    const int parts = lib.coat_grad_norm_partials((int)count, numel.data());
    if (parts < 0) check(parts, who);
    const at::Tensor work = at::empty({parts > 0 ? parts : 1}, grads[0].options().dtype(at::kDouble));
    at::Tensor out = at::empty({2}, grads[0].options().dtype(at::kFloat));
    check(lib.coat_grad_norm_multi((int)count, address.data(), kind.data(), numel.data(), (float)max_norm, (double*)work.data_ptr(), parts,
                                   (float*)out.data_ptr(), stream_of(grads[0])),
          who);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// (params, grads, exp_avg, exp_avg_sq, masters, beta1, beta2, lr, weight decay, eps, step, grad_scale) -> None.  params is not empty.
PyObject* adamw_step_multi(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    const char* who = "adamw_step_multi";
    arguments(who, n, 12);
    static const char* const names[5] = {"params", "grads", "exp_avg", "exp_avg_sq", "masters"};
    const bool masters = a[4] != Py_None;
    const int columns = masters ? 5 : 4;
    const List params(a[0], who, names[0]), grads(a[1], who, names[1]), m(a[2], who, names[2]), v(a[3], who, names[3]),
        w(masters ? a[4] : a[0], who, names[4]);
    const List* const lists[5] = {&params, &grads, &m, &v, &w};
    const Py_ssize_t count = params.size();
    TORCH_CHECK_VALUE(count > 0, who, ": no parameters");
    for (int c = 1; c < columns; c++) TORCH_CHECK(lists[c]->size() == count, who, ": the tensor lists differ in length");
    const at::Tensor* scale = tensor_or_none(a[11], who, "grad_scale");
    unrecorded(who, {scale});
    if (forward_mode())
        for (int c = 0; c < columns; c++)
            for (Py_ssize_t i = 0; i < count; i++) no_tangent((*lists[c])[i], who);
    on_gpu(params[0]);
    const at::Device device = params[0].device();
    const at::ScalarType types[5] = {params[0].scalar_type(), grads[0].scalar_type(), at::kFloat, at::kFloat, at::kFloat};
    std::vector<void*> address[5];
    std::vector<int64_t> numel(count);
    for (Py_ssize_t i = 0; i < count; i++) numel[i] = params[i].numel();
    for (int c = 0; c < columns; c++) {
        address[c].resize(count);
        for (Py_ssize_t i = 0; i < count; i++) {
            const at::Tensor& t = (*lists[c])[i];
            TORCH_CHECK(t.device() == device, who, ": ", names[c], " holds tensors that are not on the first tensor's device");
            TORCH_CHECK(t.scalar_type() == types[c], who, ": ", names[c], " must all be ", name_of(types[c]));
            TORCH_CHECK(t.numel() == numel[i], who, ": sizes of ", names[c], " differ from those of params");
            TORCH_CHECK(t.is_contiguous(), who, ": ", names[c], " must be contiguous");
            address[c][i] = t.data_ptr();
        }
    }
    const int p_dtype = code_of(types[0]), g_dtype = code_of(types[1]);
    TORCH_CHECK(g_dtype == p_dtype || g_dtype == COAT_F32, who, ": grads dtype ", name_of(types[1]), " is neither the params' ", name_of(types[0]),
                " nor torch.float32");
    TORCH_CHECK(!masters || p_dtype != COAT_F32, who, ": masters are for parameters of 16 bits");
    const int64_t step = whole(a[10]);
    TORCH_CHECK_VALUE(step >= 1 && step <= INT32_MAX, who, ": invalid step ", step);
    TORCH_CHECK(!scale || (scale->scalar_type() == at::kFloat && scale->numel() == 1 && scale->device() == device), who,
                ": grad_scale must be one fp32 element on the parameters' device");
    double hyper[5];
    for (int i = 0; i < 5; i++) hyper[i] = real(a[5 + i]);
    const c10::DeviceGuard guard(device);
    const int status = lib.coat_adamw_step_multi((int)count, address[0].data(), p_dtype, address[1].data(), g_dtype, (float**)address[2].data(),
                                                 (float**)address[3].data(), masters ? (float**)address[4].data() : nullptr, numel.data(), hyper,
                                                 (int)step, scale ? (const float*)scale->data_ptr() : nullptr, stream_of(params[0]));
    TORCH_CHECK(status != COAT_EOVERLAP, who, ": a tensor that is stepped is given twice, or shares memory with another tensor of the call");
    check(status, who);
    for (Py_ssize_t i = 0; i < count; i++)  // written behind autograd's back: graphs that saved them must notice
        if (!params[i].is_inference()) params[i].unsafeGetTensorImpl()->bump_version();
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------------ the module
// (addresses of the entry points by name, callable: device index -> stream handle)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 2 && PyDict_Check(a[0]) && PyCallable_Check(a[1]), "bind: a dictionary of addresses and a callable are needed");
#define TAKE(name)                                                             \
    {                                                                          \
        PyObject* at = PyDict_GetItemString(a[0], #name);                      \
        TORCH_CHECK_VALUE(at, "bind: no address of " #name);                   \
        lib.name = reinterpret_cast<decltype(lib.name)>(PyLong_AsVoidPtr(at)); \
        if (PyErr_Occurred()) throw python_error();                            \
        TORCH_CHECK_VALUE(lib.name, "bind: no address of " #name);             \
    }
    ENTRY_POINTS(TAKE)
#undef TAKE
    Py_XDECREF(raw_stream);
    raw_stream = Py_NewRef(a[1]);
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind),           METHOD(layer_norm_forward), METHOD(layer_norm_backward), METHOD(rotary_axes),
                         METHOD(grad_norm_multi), METHOD(adamw_step_multi),   {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddIntConstant(m, "ABI_VERSION", COAT_ABI_VERSION) != 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
