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

// A linear head: hidden [..., D], weight [V, D], bias [V] or None.
struct LinearHead {
    at::Tensor hidden, weight, bias;
    std::vector<int64_t> shape;  // of hidden
    int64_t ldh, ldw, T, D, V;
    int type;

    LinearHead(PyObject *hidden_, PyObject *weight_) : hidden(tensor("hidden", hidden_)), weight(tensor("weight", weight_))
    {
        type = checked_type("hidden", hidden);
        if (hidden.dim() < 1) refuse(PyExc_ValueError, "hidden must have the features as its last axis, is ", hidden.sizes());
        shape = hidden.sizes().vec();
        D = shape.back();
        if (weight.dim() != 2 || weight.size(1) != D)
            refuse(PyExc_ValueError, "weight must be [V, ", std::to_string(D), "], is ", weight.sizes());
        V = weight.size(0);
        if (V < 1) refuse(PyExc_ValueError, "weight must have at least one row");
        alike("weight", weight);
    }
    at::IntArrayRef tokens_of() const { return at::IntArrayRef(shape).slice(0, shape.size() - 1); }
    // the bias, and rows of the operands, of T tokens
    void settle(PyObject *bias_, int64_t tokens)
    {
        constexpr int64_t kLongestRow = 2000000;  // elements between rows that the products' 32-bit offsets reach
        if (bias_ != Py_None) {
            bias = tensor("bias", bias_);
            alike("bias", bias);
            if (bias.dim() != 1 || bias.size(0) != V)
                refuse(PyExc_ValueError, "bias must be [", std::to_string(V), "], is ", bias.sizes());
            bias = bias.contiguous();
        }
        T = tokens;
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
    const void *bias_at() const { return bias.defined() ? bias.const_data_ptr() : nullptr; }
};

// The operands of a head's cross entropy: target [...], and the number that does not count.
struct Head : LinearHead {
    at::Tensor target;
    int64_t ignore;

    explicit Head(PyObject *const *args) : LinearHead(args[0], args[1])
    {
        target = tokens("target", args[2], hidden.device());
        if (target.sizes() != tokens_of()) refuse(PyExc_ValueError, "target must be ", tokens_of(), ", is ", target.sizes());
        settle(args[3], target.numel());
        ignore = integer(args[4]);
    }

    // loss 1, gradients 2, both 3
    at::Tensor workspace(int what) const
    {
        const size_t bytes =
            ds_vocab_workspace_bytes(hidden.const_data_ptr(), ldh, weight.const_data_ptr(), ldw, T, D, V, type, what);
        return empty({(int64_t)bytes}, at::kByte);
    }
};

// The operands of a head's distillation: a teacher's ids and logits [..., K], and the temperature.
struct Pupil : LinearHead {
    at::Tensor ids, logits;
    int64_t K;
    int logits_type;
    float temperature;

    explicit Pupil(PyObject *const *args) : LinearHead(args[0], args[1])
    {
        ids = tokens("teacher_ids", args[2], hidden.device());
        if (ids.dim() < 1 || ids.sizes().slice(0, ids.dim() - 1) != tokens_of())
            refuse(PyExc_ValueError, "teacher_ids must be ", tokens_of(), " and one more axis, is ", ids.sizes());
        K = ids.size(-1);
        if (K < 1 || K > 1024) refuse(PyExc_ValueError, "a teacher must have 1 to 1024 words for a token, has ", std::to_string(K));
        logits = tensor("teacher_logits", args[3]);
        logits_type = type_code(logits);
        if (logits_type < 0)
            refuse(PyExc_TypeError, "teacher_logits must be float32, bfloat16 or float16, is ", c10::toString(logits.scalar_type()));
        if (logits.device() != hidden.device())
            refuse(PyExc_ValueError, "teacher_logits must be on ", hidden.device().str(), ", is on ", logits.device().str());
        if (logits.sizes() != ids.sizes())
            refuse(PyExc_ValueError, "teacher_logits must be ", ids.sizes(), " like teacher_ids, is ", logits.sizes());
        logits = logits.contiguous();
        int64_t tokens = 1;
        for (int64_t n : tokens_of()) tokens *= n;
        settle(args[4], tokens);
        temperature = (float)number(args[5]);
    }
    at::Tensor workspace(int what) const
    {
        return empty({(int64_t)ds_distill_workspace_bytes(hidden.const_data_ptr(), ldh, weight.const_data_ptr(), ldw, T, D, V, type,
                                                          (int)K, what)},
                     at::kByte);
    }
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

    Losses(const LinearHead &h, PyObject *red) : reduction((int)integer(red))
    {
        rows = h.empty(h.tokens_of(), at::kFloat);
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

void check_losses(const LinearHead &h, const at::Tensor &lse, const at::Tensor &grad, const at::Tensor &share)
{
    for (const at::Tensor *t : {&lse, &grad, &share})
        if (t->defined() && (t->scalar_type() != at::kFloat || !t->is_contiguous() || t->device() != h.hidden.device() ||
                             t->numel() != (t == &lse || (t == &grad && !share.defined()) ? h.T : 1)))
            refuse(PyExc_ValueError, "lse, share and grad must be float32 and fit the tokens");
}

// cross_entropy_grad(hidden, weight, target, bias or None, ignore, lse, share or None, grad, wanted, stream): gradients of
// hidden, weight and bias for `grad`, of the loss or (where there is no share) of the rows; bits 0 to 2 of `wanted` say which
PyObject *cross_entropy_grad(PyObject *, PyObject *const *args, Py_ssize_t count)
{
    return guarded(count, 10, [&] {
        const Head h(args);
        const at::Tensor &lse = tensor("lse", args[5]), &grad = tensor("grad", args[7]);
        const at::Tensor share = args[6] == Py_None ? at::Tensor() : tensor("share", args[6]);
        check_losses(h, lse, grad, share);
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

// distill(hidden, weight, teacher_ids, teacher_logits, bias or None, temperature, reduction, stream): as cross_entropy
PyObject *distill(PyObject *, PyObject *const *args, Py_ssize_t count)
{
    return guarded(count, 8, [&] {
        const Pupil h(args);
        const Losses l(h, args[6]);
        const at::Tensor ws = h.workspace(1);
        expect("ds_distill_loss",
               ds_distill_loss(h.hidden.const_data_ptr(), h.ldh, h.weight.const_data_ptr(), h.ldw, h.bias_at(),
                               h.ids.const_data_ptr(), (int)h.ids.element_size(), h.logits.const_data_ptr(), h.logits_type, (int)h.K,
                               h.temperature, h.T, h.D, h.V, h.type, l.reduction, at_or_null<float>(l.rows),
                               at_or_null<float>(l.lse), at_or_null<float>(l.total), ws.mutable_data_ptr(), ws.nbytes(),
                               stream(args[7])));
        return tuple_of({l.result(), l.lse, l.share()});
    });
}

// distill_grad(hidden, weight, teacher_ids, teacher_logits, bias or None, temperature, lse, share or None, grad, wanted, stream): as
// cross_entropy_grad
PyObject *distill_grad(PyObject *, PyObject *const *args, Py_ssize_t count)
{
    return guarded(count, 11, [&] {
        const Pupil h(args);
        const at::Tensor &lse = tensor("lse", args[6]), &grad = tensor("grad", args[8]);
        const at::Tensor share = args[7] == Py_None ? at::Tensor() : tensor("share", args[7]);
        check_losses(h, lse, grad, share);
        const int64_t wanted = integer(args[9]);
        at::Tensor dhidden, dweight, dbias;
        if (wanted & 1) dhidden = h.empty(h.shape);
        if (wanted & 2) dweight = h.empty({h.V, h.D});
        if (wanted & 4 && h.bias.defined()) dbias = h.empty({h.V});
        const at::Tensor ws = h.workspace(2);
        const float *g = (const float *)grad.const_data_ptr();
        expect("ds_distill_loss_grad",
               ds_distill_loss_grad(h.hidden.const_data_ptr(), h.ldh, h.weight.const_data_ptr(), h.ldw, h.bias_at(),
                                    h.ids.const_data_ptr(), (int)h.ids.element_size(), h.logits.const_data_ptr(), h.logits_type,
                                    (int)h.K, h.temperature, h.T, h.D, h.V, h.type, (const float *)lse.const_data_ptr(),
                                    share.defined() ? nullptr : g, share.defined() ? g : nullptr,
                                    share.defined() ? (const float *)share.const_data_ptr() : nullptr, at_or_null(dhidden),
                                    at_or_null(dweight), at_or_null(dbias), ws.mutable_data_ptr(), ws.nbytes(), stream(args[10])));
        return tuple_of({dhidden, dweight, dbias});
    });
}

// distill_step(hidden, weight, teacher_ids, teacher_logits, bias or None, temperature, reduction, stream): as cross_entropy_step
PyObject *distill_step(PyObject *, PyObject *const *args, Py_ssize_t count)
{
    return guarded(count, 8, [&] {
        const Pupil h(args);
        const Losses l(h, args[6]);
        const at::Tensor dhidden = h.empty(h.shape), dweight = h.empty({h.V, h.D});
        const at::Tensor dbias = h.bias.defined() ? h.empty({h.V}) : at::Tensor();
        const at::Tensor ws = h.workspace(3);
        expect("ds_distill_loss_step",
               ds_distill_loss_step(h.hidden.const_data_ptr(), h.ldh, h.weight.const_data_ptr(), h.ldw, h.bias_at(),
                                    h.ids.const_data_ptr(), (int)h.ids.element_size(), h.logits.const_data_ptr(), h.logits_type,
                                    (int)h.K, h.temperature, h.T, h.D, h.V, h.type, l.reduction, at_or_null<float>(l.rows),
                                    at_or_null<float>(l.lse), at_or_null<float>(l.total), at_or_null(dhidden), at_or_null(dweight),
                                    at_or_null(dbias), ws.mutable_data_ptr(), ws.nbytes(), stream(args[7])));
        return tuple_of({l.result(), dhidden, dweight, dbias});
    });
}

// Sequences [B, T, D] whose channels lie contiguously.
struct Sequences {
    at::Tensor t;
    Sequences(const at::Tensor &given) : t(given)
    {
        if (t.defined() && t.size(2) > 1 && t.stride(2) != 1) t = t.contiguous();
    }
    const void *at() const { return t.defined() ? t.const_data_ptr() : nullptr; }
    int64_t batch() const { return t.defined() && t.size(0) > 1 ? t.stride(0) : 0; }
    int64_t token() const { return t.defined() && t.size(1) > 1 ? t.stride(1) : 0; }
};

void check_like(const char *name, const at::Tensor &t, const char *like, at::ScalarType type, c10::Device device, at::IntArrayRef sizes)
{
    if (t.scalar_type() != type || t.device() != device)
        refuse(PyExc_TypeError, name, " must be ", c10::toString(type), " on ", device.str(), like, ", is ",
               c10::toString(t.scalar_type()), " on ", t.device().str());
    if (t.sizes() != sizes) refuse(PyExc_ValueError, name, " must be ", sizes, ", is ", t.sizes());
}

// The operands of a gated recurrence: x and gate [B, T, D], lengths [B] or None.
struct Recurrence {
    at::Tensor x, gate, lengths;
    int64_t B, T, D;
    int type;

    Recurrence(PyObject *x_, PyObject *gate_, PyObject *lengths_) : x(tensor("x", x_)), gate(tensor("gate", gate_))
    {
        type = checked_type("x", x);
        if (x.dim() != 3) refuse(PyExc_ValueError, "x must be [B, T, D], is ", x.sizes());
        check_like("gate", gate, " like x", x.scalar_type(), x.device(), x.sizes());
        B = x.size(0), T = x.size(1), D = x.size(2);
        if (lengths_ != Py_None) {
            lengths = tokens("lengths", lengths_, x.device());
            if (lengths.dim() != 1 || lengths.size(0) != B)
                refuse(PyExc_ValueError, "lengths must be [", std::to_string(B), "], is ", lengths.sizes());
        }
    }
    at::Tensor empty(at::IntArrayRef sizes, at::ScalarType as) const
    {
        return at::empty(sizes, at::TensorOptions().device(x.device()).dtype(as));
    }
    // float32 [B, D] or None
    at::Tensor state(const char *name, PyObject *o) const
    {
        if (o == Py_None) return at::Tensor();
        const at::Tensor &t = tensor(name, o);
        check_like(name, t, "", at::kFloat, x.device(), {B, D});
        return t.contiguous();
    }
    const void *lengths_at() const { return lengths.defined() ? lengths.const_data_ptr() : nullptr; }
    int length_bytes() const { return lengths.defined() ? (int)lengths.element_size() : 0; }
    // not defined where none is needed
    at::Tensor workspace() const
    {
        const size_t bytes = ds_recur_workspace_bytes(B, T, D, type);
        return bytes ? empty({(int64_t)bytes}, at::kByte) : at::Tensor();
    }
};

// recurrence(x, gate, state or None, lengths or None, keep, stream): all states, the last ones, and, if they are to be kept for
// gradients, those before every block
PyObject *recurrence(PyObject *, PyObject *const *args, Py_ssize_t count)
{
    return guarded(count, 6, [&] {
        const Recurrence r(args[0], args[1], args[3]);
        const at::Tensor state = r.state("state", args[2]);
        const Sequences x(r.x), gate(r.gate);
        const at::Tensor out = r.empty({r.B, r.T, r.D}, r.x.scalar_type()), last = r.empty({r.B, r.D}, at::kFloat);
        at::Tensor kept;
        if (integer(args[4])) kept = r.empty({r.B, ds_recur_blocks(r.T), r.D}, at::kFloat);
        const at::Tensor ws = r.workspace();
        expect("ds_recur_forward",
               ds_recur_forward(x.at(), x.batch(), x.token(), gate.at(), gate.batch(), gate.token(),
                                state.defined() ? (const float *)state.const_data_ptr() : nullptr, r.lengths_at(), r.length_bytes(),
                                at_or_null(out), at_or_null<float>(last), at_or_null<float>(kept), r.B, r.T, r.D, r.type,
                                at_or_null(ws), ws.defined() ? ws.nbytes() : 0, stream(args[5])));
        return tuple_of({out, last, kept});
    });
}

// recurrence_grad(x, gate, grad or None, grad_last or None, lengths or None, kept, wanted, stream): gradients of x, gate and the
// first state; bits 0 to 2 of `wanted` say which
PyObject *recurrence_grad(PyObject *, PyObject *const *args, Py_ssize_t count)
{
    return guarded(count, 8, [&] {
        const Recurrence r(args[0], args[1], args[4]);
        const at::Tensor grad_last = r.state("grad_last", args[3]);
        const at::Tensor given = args[2] == Py_None ? at::Tensor() : tensor("grad", args[2]);
        if (given.defined()) check_like("grad", given, " like x", r.x.scalar_type(), r.x.device(), r.x.sizes());
        const at::Tensor &kept = tensor("kept", args[5]);
        check_like("kept", kept, "", at::kFloat, r.x.device(), {r.B, ds_recur_blocks(r.T), r.D});
        const Sequences x(r.x), gate(r.gate), grad(given);
        const int64_t wanted = integer(args[6]);
        at::Tensor dx, dgate, dstate;
        if (wanted & 1) dx = r.empty(r.x.sizes(), r.x.scalar_type());
        if (wanted & 2) dgate = r.empty(r.x.sizes(), r.x.scalar_type());
        if (wanted & 4) dstate = r.empty({r.B, r.D}, at::kFloat);
        const at::Tensor ws = r.workspace();
        expect("ds_recur_backward",
               ds_recur_backward(x.at(), x.batch(), x.token(), gate.at(), gate.batch(), gate.token(), grad.at(), grad.batch(),
                                 grad.token(), grad_last.defined() ? (const float *)grad_last.const_data_ptr() : nullptr,
                                 r.lengths_at(), r.length_bytes(), (const float *)kept.contiguous().const_data_ptr(), at_or_null(dx),
                                 at_or_null(dgate), at_or_null<float>(dstate), r.B, r.T, r.D, r.type, at_or_null(ws),
                                 ws.defined() ? ws.nbytes() : 0, stream(args[7])));
        return tuple_of({dx, dgate, dstate});
    });
}

// The operands of a gated block: x [..., D], weight [2 F, D], bias [2 F] or None.
struct Gated {
    at::Tensor x, weight, bias;
    std::vector<int64_t> shape;  // of x
    int64_t ldx, ldw, T, D, F, activation;
    int type;

    Gated(PyObject *x_, PyObject *weight_, PyObject *bias_, PyObject *activation_) : x(tensor("x", x_)), weight(tensor("weight", weight_))
    {
        constexpr int64_t kLongestRow = 2000000;
        type = checked_type("x", x);
        if (x.dim() < 1) refuse(PyExc_ValueError, "x must have the features as its last axis, is ", x.sizes());
        shape = x.sizes().vec();
        D = shape.back();
        if (weight.dim() != 2 || weight.size(1) != D || weight.size(0) % 2)
            refuse(PyExc_ValueError, "weight must be [2 F, ", std::to_string(D), "], is ", weight.sizes());
        F = weight.size(0) / 2;
        check_like("weight", weight, " like x", x.scalar_type(), x.device(), weight.sizes());
        if (bias_ != Py_None) {
            bias = tensor("bias", bias_);
            check_like("bias", bias, " like x", x.scalar_type(), x.device(), {2 * F});
            bias = bias.contiguous();
        }
        activation = integer(activation_);
        T = 1;
        for (size_t i = 0; i + 1 < shape.size(); ++i) T *= shape[i];
        if (x.dim() != 2) x = x.reshape({T, D});
        ldx = rows(x, kLongestRow);
        ldw = rows(weight, kLongestRow);
    }
    at::Tensor empty(at::IntArrayRef sizes, at::ScalarType as) const
    {
        return at::empty(sizes, at::TensorOptions().device(x.device()).dtype(as));
    }
    at::Tensor empty(at::IntArrayRef sizes) const { return empty(sizes, x.scalar_type()); }
    at::Tensor workspace(int what) const
    {
        return empty({(int64_t)ds_gated_workspace_bytes(x.const_data_ptr(), ldx, weight.const_data_ptr(), ldw, T, D, F, type, what)},
                     at::kByte);
    }
    std::vector<int64_t> kept() const { return {T, 2, (F + 7) / 8 * 8}; }
};

// gated(x, weight, bias or None, activation, keep, stream): the block's result, and both halves of its product if they are to be
// kept for gradients
PyObject *gated(PyObject *, PyObject *const *args, Py_ssize_t count)
{
    return guarded(count, 6, [&] {
        const Gated g(args[0], args[1], args[2], args[3]);
        std::vector<int64_t> shape = g.shape;
        shape.back() = g.F;
        const at::Tensor out = g.empty(shape);
        at::Tensor halves;
        if (integer(args[4])) halves = g.empty(g.kept(), at::kFloat);
        const at::Tensor ws = g.workspace(1);
        expect("ds_gated_forward",
               ds_gated_forward(g.x.const_data_ptr(), g.ldx, g.weight.const_data_ptr(), g.ldw,
                                g.bias.defined() ? g.bias.const_data_ptr() : nullptr, (int)g.activation, g.T, g.D, g.F, g.type,
                                at_or_null(out), at_or_null<float>(halves), ws.mutable_data_ptr(), ws.nbytes(), stream(args[5])));
        return tuple_of({out, halves});
    });
}

// gated_grad(x, weight, halves, grad, activation, wanted, stream): gradients of x, weight and bias; bits 0 to 2 of `wanted` say
// which
PyObject *gated_grad(PyObject *, PyObject *const *args, Py_ssize_t count)
{
    return guarded(count, 7, [&] {
        const Gated g(args[0], args[1], Py_None, args[4]);
        const at::Tensor &halves = tensor("halves", args[2]);
        check_like("halves", halves, "", at::kFloat, g.x.device(), g.kept());
        at::Tensor grad = tensor("grad", args[3]);
        std::vector<int64_t> shape = g.shape;
        shape.back() = g.F;
        check_like("grad", grad, " like x", g.x.scalar_type(), g.x.device(), shape);
        if (grad.dim() != 2) grad = grad.reshape({g.T, g.F});
        const int64_t ldg = rows(grad), wanted = integer(args[5]);
        at::Tensor dx, dweight, dbias;
        if (wanted & 1) dx = g.empty(g.shape);
        if (wanted & 2) dweight = g.empty({2 * g.F, g.D});
        if (wanted & 4) dbias = g.empty({2 * g.F});
        const at::Tensor ws = g.workspace(2);
        expect("ds_gated_backward",
               ds_gated_backward(g.x.const_data_ptr(), g.ldx, g.weight.const_data_ptr(), g.ldw, (const float *)halves.const_data_ptr(),
                                 grad.const_data_ptr(), ldg, (int)g.activation, g.T, g.D, g.F, g.type, at_or_null(dx),
                                 at_or_null(dweight), at_or_null(dbias), ws.mutable_data_ptr(), ws.nbytes(), stream(args[6])));
        return tuple_of({dx, dweight, dbias});
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
    {"distill", (PyCFunction)(void (*)(void))distill, METH_FASTCALL,
     "distill(hidden, weight, teacher_ids, teacher_logits, bias or None, temperature, reduction, stream) -> loss, lse, share or None"},
    {"distill_grad", (PyCFunction)(void (*)(void))distill_grad, METH_FASTCALL,
     "distill_grad(hidden, weight, teacher_ids, teacher_logits, bias or None, temperature, lse, share or None, grad, wanted, stream) "
     "-> gradients"},
    {"distill_step", (PyCFunction)(void (*)(void))distill_step, METH_FASTCALL,
     "distill_step(hidden, weight, teacher_ids, teacher_logits, bias or None, temperature, reduction, stream) -> loss, gradients"},
    {"recurrence", (PyCFunction)(void (*)(void))recurrence, METH_FASTCALL,
     "recurrence(x, gate, state or None, lengths or None, keep, stream) -> states, last ones, kept ones or None"},
    {"recurrence_grad", (PyCFunction)(void (*)(void))recurrence_grad, METH_FASTCALL,
     "recurrence_grad(x, gate, grad or None, grad_last or None, lengths or None, kept, wanted, stream) -> gradients"},
    {"gated", (PyCFunction)(void (*)(void))gated, METH_FASTCALL,
     "gated(x, weight, bias or None, activation, keep, stream) -> result, halves of the product or None"},
    {"gated_grad", (PyCFunction)(void (*)(void))gated_grad, METH_FASTCALL,
     "gated_grad(x, weight, halves, grad, activation, wanted, stream) -> gradients"},
    {"clip", (PyCFunction)(void (*)(void))clip, METH_FASTCALL,
     "clip(grads, outs or None, max_norm, scale, any_order, stream) -> norm, or None"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ds_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_ds_torch(void) { return PyModule_Create(&module); }
