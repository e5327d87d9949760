// The host's side of a training step's operators, whose kernels may be over sooner than a few dozen steps of the Python
// interpreter: checks, allocations and the call of the library, on torch's tensors as they are.
//
// Bound by the launches themselves (2.7 us each) and torch's allocations (0.8 us).
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/TracerMode.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <algorithm>
#include <string>
#include <vector>
#include "deepshift_hip.h"

namespace {

// What a caller hears: the type of a Python exception and its text.
struct Refusal {
    PyObject *type;
    std::string text;
};

struct Failure {
    const char *entry;
    int status;
};

int type_code(const at::Tensor &t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return DS_F32;
    case at::kBFloat16: return DS_BF16;
    case at::kHalf: return DS_F16;
    default: return -1;
    }
}

std::string text_of(const char *what) { return what; }
std::string text_of(const std::string &what) { return what; }
std::string text_of(at::IntArrayRef sizes)
{
    std::string s = "[";
    for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
    return s + "]";
}
template <typename... T> [[noreturn]] void refuse(PyObject *type, const T &...parts) { throw Refusal{type, (text_of(parts) + ...)}; }

const at::Tensor &tensor(const char *name, PyObject *o)
{
    if (!THPVariable_Check(o)) refuse(PyExc_TypeError, name, " must be a tensor, is ", Py_TYPE(o)->tp_name);
    const at::Tensor &t = THPVariable_Unpack(o);
    if (t._fw_grad(0).defined())
        refuse(PyExc_NotImplementedError, name, " has a tangent, and these operators have no forward-mode derivatives");
    if (t.is_neg()) refuse(PyExc_ValueError, name, " is a lazily negated view: resolve_neg() gives its values");
    return t;
}

int checked_type(const char *name, const at::Tensor &t)
{
    const int code = type_code(t);
    if (code < 0) refuse(PyExc_TypeError, name, " must be float32, bfloat16 or float16, is ", c10::toString(t.scalar_type()));
    if (!t.is_cuda()) refuse(PyExc_ValueError, name, " must be a GPU tensor");
    return code;
}

int64_t integer(PyObject *o)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refusal{nullptr, ""};
    return v;
}
double number(PyObject *o)
{
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Refusal{nullptr, ""};
    return v;
}
void *stream(PyObject *o)
{
    void *p = PyLong_AsVoidPtr(o);
    if (!p && PyErr_Occurred()) throw Refusal{nullptr, ""};
    return p;
}

void expect(const char *entry, int status)
{
    if (status != DS_OK) throw Failure{entry, status};
}

// A trace would hold the allocation of a result, and nothing that writes it.
void refuse_tracing()
{
    namespace modes = c10::impl;
    if (at::tracer::impl::is_dispatch_enabled() ||
        (modes::TorchDispatchModeTLS::any_modes_set() &&
         modes::TorchDispatchModeTLS::get_mode(modes::TorchDispatchModeKey::PROXY).has_value()))
        refuse(PyExc_NotImplementedError, "these operators cannot be traced");
}

// Runs an entry point; whatever is thrown in it becomes a Python exception.
template <typename F> PyObject *guarded(Py_ssize_t got, Py_ssize_t wanted, F &&body)
{
    try {
        if (got != wanted) refuse(PyExc_TypeError, std::to_string(wanted), " arguments expected");
        refuse_tracing();
        return body();
    } catch (const Refusal &r) {
        if (r.type) PyErr_SetString(r.type, r.text.c_str());
    } catch (const Failure &f) {
        PyObject *module = PyImport_ImportModule("deepshift_amd._lib");
        PyObject *type = module ? PyObject_GetAttrString(module, "DeepShiftError") : nullptr;
        PyObject *args = type ? Py_BuildValue("(sis)", f.entry, f.status, ds_status_string(f.status)) : nullptr;
        if (args) PyErr_SetObject(type, args);
        Py_XDECREF(args);
        Py_XDECREF(type);
        Py_XDECREF(module);
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

// Token numbers on a device, contiguous.
at::Tensor tokens(const char *name, PyObject *o, c10::Device device)
{
    const at::Tensor &ids = tensor(name, o);
    if (ids.scalar_type() != at::kLong && ids.scalar_type() != at::kInt)
        refuse(PyExc_TypeError, name, " must be int64 or int32, is ", c10::toString(ids.scalar_type()));
    if (ids.device() != device) refuse(PyExc_ValueError, name, " must be on ", device.str(), ", is on ", ids.device().str());
    return ids.is_contiguous() ? ids : ids.contiguous();
}

// A matrix whose rows lie contiguously, up to `most` elements apart, and their distance.
int64_t rows(at::Tensor &t, int64_t most = INT64_MAX)
{
    const int64_t n = t.size(0), D = t.size(1);
    if ((D > 1 && t.stride(1) != 1) || (n > 1 && (t.stride(0) < D || t.stride(0) > most))) t = t.contiguous();
    return n > 1 ? t.stride(0) : D;
}

// embed(ids, weight, scale, stream): scale * weight[ids]
PyObject *embed(PyObject *, PyObject *const *args, Py_ssize_t count)
{
    return guarded(count, 4, [&] {
        at::Tensor weight = tensor("weight", args[1]);
        const int code = checked_type("weight", weight);
        if (weight.dim() != 2) refuse(PyExc_ValueError, "weight must be [V, D], is ", weight.sizes());
        const at::Tensor ids = tokens("ids", args[0], weight.device());
        const int64_t V = weight.size(0), D = weight.size(1), ld = rows(weight);
        c10::SmallVector<int64_t, 6> shape(ids.sizes().begin(), ids.sizes().end());
        shape.push_back(D);
        at::Tensor out = at::empty(shape, weight.options().requires_grad(false));
        expect("ds_embed", ds_embed(ids.const_data_ptr(), (int)ids.element_size(), weight.const_data_ptr(), ld,
                                    out.mutable_data_ptr(), ids.numel(), V, D, (float)number(args[2]), code, stream(args[3])));
        return THPVariable_Wrap(std::move(out));
    });
}

// embed_grad(ids, grad, V, scale, padding, stream): the gradient of embed with respect to a weight of V rows
PyObject *embed_grad(PyObject *, PyObject *const *args, Py_ssize_t count)
{
    return guarded(count, 6, [&] {
        const at::Tensor &given = tensor("grad", args[1]);
        const int code = checked_type("grad", given);
        const at::Tensor ids = tokens("ids", args[0], given.device());
        if (given.dim() < 1 || given.sizes().slice(0, given.dim() - 1) != ids.sizes())
            refuse(PyExc_ValueError, "grad must have the shape of ids, ", ids.sizes(), ", and one more axis, is ", given.sizes());
        const int64_t T = ids.numel(), D = given.size(-1), V = integer(args[2]);
        if (V < 0) refuse(PyExc_ValueError, "num_embeddings must not be negative");
        at::Tensor grad = given.reshape({T, D});
        const int64_t ld = rows(grad);
        const at::TensorOptions options = grad.options().requires_grad(false);
        at::Tensor out = at::empty({V, D}, options);
        const size_t bytes = ds_embed_grad_workspace_bytes(T, D);
        at::Tensor workspace = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
        expect("ds_embed_grad", ds_embed_grad(ids.const_data_ptr(), (int)ids.element_size(), grad.const_data_ptr(), ld,
                                              out.mutable_data_ptr(), T, V, D, integer(args[4]), (float)number(args[3]), code,
                                              workspace.mutable_data_ptr(), bytes, stream(args[5])));
        return THPVariable_Wrap(std::move(out));
    });
}

// The operands of a head's cross entropy: hidden [..., D], weight [V, D], target [...], bias [V] or None.
struct Head {
    at::Tensor hidden, weight, target, bias;
    std::vector<int64_t> shape;  // of hidden
    int64_t ldh, ldw, T, D, V, ignore;
    int type;

    explicit Head(PyObject *const *args) : hidden(tensor("hidden", args[0])), weight(tensor("weight", args[1]))
    {
        constexpr int64_t kLongestRow = 2000000;  // elements between rows that the products' 32-bit offsets reach
        type = checked_type("hidden", hidden);
        if (hidden.dim() < 1) refuse(PyExc_ValueError, "hidden must have the features as its last axis, is ", hidden.sizes());
        shape = hidden.sizes().vec();
        D = shape.back();
        if (weight.dim() != 2 || weight.size(1) != D)
            refuse(PyExc_ValueError, "weight must be [V, ", std::to_string(D), "], is ", weight.sizes());
        V = weight.size(0);
        if (V < 1) refuse(PyExc_ValueError, "weight must have at least one row");
        alike("weight", weight);
        target = tokens("target", args[2], hidden.device());
        if (target.sizes() != hidden.sizes().slice(0, shape.size() - 1))
            refuse(PyExc_ValueError, "target must be ", hidden.sizes().slice(0, shape.size() - 1), ", is ", target.sizes());
        if (args[3] != Py_None) {
            bias = tensor("bias", args[3]);
            alike("bias", bias);
            if (bias.dim() != 1 || bias.size(0) != V)
                refuse(PyExc_ValueError, "bias must be [", std::to_string(V), "], is ", bias.sizes());
            bias = bias.contiguous();
        }
        ignore = integer(args[4]);
        T = target.numel();
        if (hidden.dim() != 2) hidden = hidden.reshape({T, D});
        ldh = rows(hidden, kLongestRow);
        ldw = rows(weight, kLongestRow);
    }

    void alike(const char *name, const at::Tensor &t) const
    {
        if (t.scalar_type() != hidden.scalar_type() || t.device() != hidden.device())
            refuse(PyExc_TypeError, name, " must be ", c10::toString(hidden.scalar_type()), " on ", hidden.device().str(),
                   " like hidden, is ", c10::toString(t.scalar_type()), " on ", t.device().str());
    }

    at::Tensor empty(at::IntArrayRef sizes, at::ScalarType as) const
    {
        return at::empty(sizes, at::TensorOptions().device(hidden.device()).dtype(as));
    }
    at::Tensor empty(at::IntArrayRef sizes) const { return empty(sizes, hidden.scalar_type()); }

    // loss 1, gradients 2, both 3
    at::Tensor workspace(int what) const
    {
        const size_t bytes =
            ds_vocab_workspace_bytes(hidden.const_data_ptr(), ldh, weight.const_data_ptr(), ldw, T, D, V, type, what);
        return empty({(int64_t)bytes}, at::kByte);
    }
    const void *bias_at() const { return bias.defined() ? bias.const_data_ptr() : nullptr; }
};

template <typename E = void> E *at_or_null(const at::Tensor &t) { return t.defined() ? (E *)t.mutable_data_ptr() : nullptr; }

// New references to tensors, None for those that are not defined.
PyObject *tuple_of(std::initializer_list<at::Tensor> tensors)
{
    PyObject *t = PyTuple_New((Py_ssize_t)tensors.size());
    if (!t) return nullptr;
    Py_ssize_t i = 0;
    for (const at::Tensor &x : tensors) PyTuple_SET_ITEM(t, i++, THPVariable_Wrap(x));
    return t;
}

// A scalar of its own on element `i` of `t`'s memory: what a Function returns may be changed in place (loss /= n), unless it is a
// view, and counts its changes by itself.
at::Tensor scalar_at(const at::Tensor &t, int64_t i)
{
    at::Tensor s = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(), t.dtype());
    s.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef{}, at::IntArrayRef{}, t.storage_offset() + i);
    return s;
}

// What a call finds out about the losses of rows.
struct Losses {
    int reduction;
    at::Tensor rows, lse, total;

    Losses(const Head &h, PyObject *red) : reduction((int)integer(red))
    {
        rows = h.empty(h.target.sizes(), at::kFloat);
        lse = h.empty({h.T}, at::kFloat);
        if (reduction) total = h.empty({2}, at::kFloat);
    }
    at::Tensor result() const { return reduction ? scalar_at(total, 0) : rows; }
    at::Tensor share() const { return reduction ? scalar_at(total, 1) : at::Tensor(); }
};

// cross_entropy(hidden, weight, target, bias or None, ignore, reduction, stream): the loss, and what its gradients need: the
// rows' logarithms, and a row's share in the loss where it is reduced
PyObject *cross_entropy(PyObject *, PyObject *const *args, Py_ssize_t count)
{
    return guarded(count, 7, [&] {
        const Head h(args);
        const Losses l(h, args[5]);
        const at::Tensor ws = h.workspace(1);
        expect("ds_vocab_loss",
               ds_vocab_loss(h.hidden.const_data_ptr(), h.ldh, h.weight.const_data_ptr(), h.ldw, h.bias_at(),
                             h.target.const_data_ptr(), (int)h.target.element_size(), h.ignore, h.T, h.D, h.V, h.type, l.reduction,
                             at_or_null<float>(l.rows), at_or_null<float>(l.lse), at_or_null<float>(l.total),
                             ws.mutable_data_ptr(), ws.nbytes(), stream(args[6])));
        return tuple_of({l.result(), l.lse, l.share()});
    });
}

// cross_entropy_grad(hidden, weight, target, bias or None, ignore, lse, share or None, grad, wanted, stream): gradients of
// hidden, weight and bias for `grad`, of the loss or (where there is no share) of the rows; bits 0 to 2 of `wanted` say which
PyObject *cross_entropy_grad(PyObject *, PyObject *const *args, Py_ssize_t count)
{
    return guarded(count, 10, [&] {
        const Head h(args);
        const at::Tensor &lse = tensor("lse", args[5]), &grad = tensor("grad", args[7]);
        const at::Tensor share = args[6] == Py_None ? at::Tensor() : tensor("share", args[6]);
        for (const at::Tensor *t : {&lse, &grad, &share})
            if (t->defined() && (t->scalar_type() != at::kFloat || !t->is_contiguous() || t->device() != h.hidden.device() ||
                                 t->numel() != (t == &lse || (t == &grad && !share.defined()) ? h.T : 1)))
                refuse(PyExc_ValueError, "lse, share and grad must be float32 and fit the tokens");
        const int64_t wanted = integer(args[8]);
        at::Tensor dhidden, dweight, dbias;
        if (wanted & 1) dhidden = h.empty(h.shape);
        if (wanted & 2) dweight = h.empty({h.V, h.D});
        if (wanted & 4 && h.bias.defined()) dbias = h.empty({h.V});
        const at::Tensor ws = h.workspace(2);
        const float *g = (const float *)grad.const_data_ptr();
        expect("ds_vocab_loss_grad",
               ds_vocab_loss_grad(h.hidden.const_data_ptr(), h.ldh, h.weight.const_data_ptr(), h.ldw, h.bias_at(),
                                  h.target.const_data_ptr(), (int)h.target.element_size(), h.ignore, h.T, h.D, h.V, h.type,
                                  (const float *)lse.const_data_ptr(), share.defined() ? nullptr : g, share.defined() ? g : nullptr,
                                  share.defined() ? (const float *)share.const_data_ptr() : nullptr, at_or_null(dhidden),
                                  at_or_null(dweight), at_or_null(dbias), ws.mutable_data_ptr(), ws.nbytes(), stream(args[9])));
        return tuple_of({dhidden, dweight, dbias});
    });
}

// cross_entropy_step(hidden, weight, target, bias or None, ignore, reduction, stream): the loss and its gradients, for a
// gradient of 1
PyObject *cross_entropy_step(PyObject *, PyObject *const *args, Py_ssize_t count)
{
    return guarded(count, 7, [&] {
        const Head h(args);
        const Losses l(h, args[5]);
        const at::Tensor dhidden = h.empty(h.shape), dweight = h.empty({h.V, h.D});
        const at::Tensor dbias = h.bias.defined() ? h.empty({h.V}) : at::Tensor();
        const at::Tensor ws = h.workspace(3);
        expect("ds_vocab_loss_step",
               ds_vocab_loss_step(h.hidden.const_data_ptr(), h.ldh, h.weight.const_data_ptr(), h.ldw, h.bias_at(),
                                  h.target.const_data_ptr(), (int)h.target.element_size(), h.ignore, h.T, h.D, h.V, h.type,
                                  l.reduction, at_or_null<float>(l.rows), at_or_null<float>(l.lse), at_or_null<float>(l.total),
                                  at_or_null(dhidden), at_or_null(dweight), at_or_null(dbias), ws.mutable_data_ptr(), ws.nbytes(),
                                  stream(args[6])));
        return tuple_of({l.result(), dhidden, dweight, dbias});
    });
}

// The tensors of a list: types, one device; false where one is not contiguous.
bool look_at(const char *name, PyObject *list, c10::Device device, std::vector<const at::Tensor *> &tensors, std::vector<int> &types)
{
    bool contiguous = true;
    const Py_ssize_t n = PyList_GET_SIZE(list);
    tensors.reserve(n), types.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
        const at::Tensor &t = tensor(name, PyList_GET_ITEM(list, i));
        types.push_back(checked_type(name, t));
        if (t.device() != device) refuse(PyExc_ValueError, "every ", name, " must be on one device, the first gradient's");
        contiguous = t.is_contiguous() && contiguous;
        tensors.push_back(&t);
    }
    return contiguous;
}

int64_t bytes_of(int64_t n, int type) { return n * (type == DS_F32 ? 4 : 2); }

// Nothing may be written twice, and what one tensor's elements are read from may not be written for another: workgroups do both at
// the same time.  A tensor scaled in place, to its own type, is read by whoever writes it.
void check_overlaps(const std::vector<ds_tensor> &table)
{
    struct Range {
        uintptr_t from, to;
        bool written;
        bool operator<(const Range &o) const { return from < o.from; }
    };
    std::vector<Range> ranges;
    ranges.reserve(2 * table.size());
    for (const ds_tensor &x : table) {
        if (x.n == 0) continue;
        ranges.push_back({(uintptr_t)x.dst, (uintptr_t)x.dst + bytes_of(x.n, x.dst_type), true});
        if (x.src != x.dst || x.src_type != x.dst_type)
            ranges.push_back({(uintptr_t)x.src, (uintptr_t)x.src + bytes_of(x.n, x.src_type), false});
    }
    if (!std::is_sorted(ranges.begin(), ranges.end())) std::sort(ranges.begin(), ranges.end());
    uintptr_t any = 0, written = 0;  // where the ranges so far end at the latest
    for (const Range &r : ranges) {
        if (r.from < (r.written ? any : written))
            refuse(PyExc_ValueError, "a tensor is given twice, or one that is written shares memory with another one");
        any = std::max(any, r.to);
        if (r.written) written = std::max(written, r.to);
    }
}

// clip(grads, outs or None, max_norm, scale, any_order, stream): the norm; None, with nothing done, where a tensor is not
// contiguous and the caller has not said by `any_order` that all elements fill stretches of memory in the same order.
PyObject *clip(PyObject *, PyObject *const *args, Py_ssize_t count)
{
    return guarded(count, 6, [&]() -> PyObject * {
        PyObject *const grads = args[0], *const outs = args[1];
        if (!PyList_Check(grads) || (outs != Py_None && !PyList_Check(outs))) refuse(PyExc_TypeError, "lists of tensors expected");
        const Py_ssize_t n = PyList_GET_SIZE(grads);
        if (n == 0 || n > 0x7fffffff) refuse(PyExc_ValueError, n ? "too many gradients" : "no gradients given");
        const bool elsewhere = outs != Py_None, scale = integer(args[3]) != 0, any_order = integer(args[4]) != 0;
        if (elsewhere && PyList_GET_SIZE(outs) != n)
            refuse(PyExc_ValueError, std::to_string(PyList_GET_SIZE(outs)), " tensors in out for ", std::to_string(n), " gradients");
        std::vector<const at::Tensor *> from, to_elsewhere;
        std::vector<int> from_types, to_types;
        const c10::Device device = tensor("gradient", PyList_GET_ITEM(grads, 0)).device();
        bool contiguous = look_at("gradient", grads, device, from, from_types);
        if (elsewhere) {
            contiguous = look_at("out", outs, device, to_elsewhere, to_types) && contiguous;
            for (Py_ssize_t i = 0; i < n; ++i)
                if (from[i]->sizes() != to_elsewhere[i]->sizes())
                    refuse(PyExc_ValueError, "out ", std::to_string(i), " must be ", from[i]->sizes(), ", is ",
                           to_elsewhere[i]->sizes());
        }
        if (!contiguous && !any_order) Py_RETURN_NONE;
        const std::vector<const at::Tensor *> &to = elsewhere ? to_elsewhere : from;

        std::vector<ds_tensor> table(n);
        for (Py_ssize_t i = 0; i < n; ++i) {
            ds_tensor &x = table[i];
            x.src = from[i]->const_data_ptr();
            x.dst = scale ? to[i]->mutable_data_ptr() : const_cast<void *>(x.src);
            // (a tensor that shares its memory until it is written to has moved)
            if (scale && !elsewhere) x.src = x.dst;
            x.n = from[i]->numel();
            x.src_type = from_types[i], x.dst_type = elsewhere ? to_types[i] : from_types[i];
        }
        if (scale) check_overlaps(table);
        const auto options = at::TensorOptions().device(device);
        at::Tensor norm = at::empty({}, options.dtype(at::kFloat));
        const size_t bytes = ds_clip_workspace_bytes((int)n);
        at::Tensor workspace = at::empty({(int64_t)bytes}, options.dtype(at::kByte));
        expect("ds_clip", ds_clip(table.data(), (int)n, (float)number(args[2]), scale, (float *)norm.mutable_data_ptr(),
                                  workspace.mutable_data_ptr(), bytes, stream(args[5])));
        // autograd hears of what was written behind its back; inference tensors keep no count
        if (scale)
            for (const at::Tensor *t : to)
                if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
        return THPVariable_Wrap(std::move(norm));
    });
}

PyMethodDef methods[] = {
    {"embed", (PyCFunction)(void (*)(void))embed, METH_FASTCALL, "embed(ids, weight, scale, stream) -> scale * weight[ids]"},
    {"embed_grad", (PyCFunction)(void (*)(void))embed_grad, METH_FASTCALL,
     "embed_grad(ids, grad, V, scale, padding, stream) -> gradient of a weight of V rows"},
    {"cross_entropy", (PyCFunction)(void (*)(void))cross_entropy, METH_FASTCALL,
     "cross_entropy(hidden, weight, target, bias or None, ignore, reduction, stream) -> loss, lse, share or None"},
    {"cross_entropy_grad", (PyCFunction)(void (*)(void))cross_entropy_grad, METH_FASTCALL,
     "cross_entropy_grad(hidden, weight, target, bias or None, ignore, lse, share or None, grad, wanted, stream) -> gradients"},
    {"cross_entropy_step", (PyCFunction)(void (*)(void))cross_entropy_step, METH_FASTCALL,
     "cross_entropy_step(hidden, weight, target, bias or None, ignore, reduction, stream) -> loss, gradients"},
    {"clip", (PyCFunction)(void (*)(void))clip, METH_FASTCALL,
     "clip(grads, outs or None, max_norm, scale, any_order, stream) -> norm, or None"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ds_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_ds_torch(void) { return PyModule_Create(&module); }
