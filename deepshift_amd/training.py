"""Operators of a token model's training step around shift layers: the scaled embedding lookup at its entrance, the gated
recurrence that mixes a sequence's tokens and the gated block of a feed-forward layer between, the cross entropy of a linear head
over a large vocabulary, and its distance from a teacher's best words, at its exit, and the clipping of gradients by their global
norm.

The layers between are ``LinearShift`` / ``LinearShiftQ`` on their float path, whose straight-through gradients
(``ste.py``) reach shifts and signs unscaled -- the reason to clip them.  Everything here runs in the gfx950 library, on the
current stream of the tensors' device, on float32, bfloat16 and float16; sums are held in 32 bits or more and rounded once,
and a call repeats bit for bit.  In 16-bit types the matrix instructions take gradients in that type too: probabilities of a
vocabulary, and the gradient of a gated block's projections, are rounded to it before the products that they go into (but for
:func:`linear_distillation`'s frequent words in bfloat16, which keep what that loses).  There is no CPU path: a CPU tensor raises.

Functions whose names end in ``_grad`` return gradients directly; the others, but for the clipping, take part in autograd.  All
can be captured into a graph; where ``backward()`` is, no graph recorded eagerly from the same parameters may be alive (PyTorch
adds gradients up on the stream that recorded them first).
"""
import contextlib

import torch
import torch.nn as nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib, modules, modules_q

__all__ = ["embedding", "embedding_grad", "linear_cross_entropy", "linear_cross_entropy_grad", "linear_distillation",
           "linear_distillation_grad", "gated_linear", "gated_recurrence", "gradient_norm", "clip_gradients_", "clip_grad_norm_",
           "ScaledEmbedding", "LinearCrossEntropy", "GatedLinear", "GatedShift"]

_REDUCTIONS = {"none": _lib.DS_NONE, "sum": _lib.DS_SUM, "mean": _lib.DS_MEAN}


_HERE = contextlib.nullcontext()


def _on(device):
    """Makes a tensor's device the current one for the launches of a call."""
    if device.type != "cuda" or device.index == torch._C._cuda_getDevice():
        return _HERE
    return torch.cuda.device(device)


def _stream_of(device):
    return _lib.stream_handle(device) if device.type == "cuda" else 0   # a CPU tensor is refused further down


# ---------------------------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------------------------

def _embed(ids, weight, scale):
    device = weight.device
    with _on(device):
        return _lib.native().embed(ids, weight, scale, _stream_of(device))


def embedding_grad(ids, grad, num_embeddings, scale=1.0, padding_idx=None):
    """Gradient of :func:`embedding` with respect to its weight, ``[num_embeddings, D]`` in ``grad``'s type: row ``v`` is
    ``scale`` times the sum of ``grad`` over the tokens ``v``, in ascending order and 32 bits.  Tokens equal to
    ``padding_idx`` add nothing, and neither do numbers outside ``[0, num_embeddings)``."""
    V, scale = int(num_embeddings), _scale(scale)
    padding = _padding(padding_idx, V)
    device = grad.device
    with _on(device):
        return _lib.native().embed_grad(ids, grad, V, scale, padding, _stream_of(device))


_LARGEST = (2 - 2.0 ** -24) * 2.0 ** 127   # float32 rounds it, and what is beyond, to infinity


def _scale(scale):
    scale = float(scale)
    if not abs(scale) < _LARGEST:
        raise ValueError("scale must be finite in float32, is %r" % scale)
    return scale


def _padding(padding_idx, V):
    if padding_idx is None:
        return -1
    if not -V <= padding_idx < V:
        raise ValueError("padding_idx must be in [-%d, %d), is %d" % (V, V, padding_idx))
    return padding_idx % V


class _Embedding(Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.of = (weight.shape[0], scale, padding_idx)
        return _embed(ids, weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        V, scale, padding_idx = ctx.of
        return None, embedding_grad(ids, grad, V, scale, padding_idx), None, None


def embedding(ids, weight, scale=1.0, padding_idx=None):
    """``scale * weight[ids]`` for ``ids`` of any shape (int64 or int32) and ``weight`` ``[V, D]``, multiplied in 32 bits and
    rounded once.  A number outside ``[0, V)`` gives a row of NaN (the GPU cannot raise).  ``padding_idx`` names the word
    whose row gets no gradient."""
    scale = _scale(scale)
    if padding_idx is not None and weight.dim() == 2:
        _padding(padding_idx, weight.shape[0])
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(ids, weight, scale, padding_idx)
    return _embed(ids, weight, scale)


# ---------------------------------------------------------------------------------------------
# cross entropy of a linear head
# ---------------------------------------------------------------------------------------------

def _decided(ignore_index, reduction):
    """``ignore_index`` and ``reduction`` as the library takes them."""
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction must be 'none', 'sum' or 'mean', is %r" % (reduction,))
    ignore_index = int(ignore_index)
    if not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError("ignore_index must fit 64 bits")
    return ignore_index, _REDUCTIONS[reduction]


class _LinearCrossEntropy(Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, bias, ignore_index, reduction):
        device = hidden.device
        with _on(device):
            loss, lse, share = _lib.native().cross_entropy(hidden, weight, target, bias, ignore_index, reduction,
                                                           _stream_of(device))
        ctx.save_for_backward(hidden, weight, target, bias, lse, share)
        ctx.ignore_index = ignore_index
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        hidden, weight, target, bias, lse, share = ctx.saved_tensors
        device, needed = hidden.device, ctx.needs_input_grad
        with _on(device):
            dhidden, dweight, dbias = _lib.native().cross_entropy_grad(
                hidden, weight, target, bias, ctx.ignore_index, lse, share, grad.float().contiguous(),
                needed[0] | needed[1] << 1 | needed[3] << 2, _stream_of(device))
        return dhidden, dweight, None, dbias, None, None


def linear_cross_entropy(hidden, weight, target, bias=None, ignore_index=-100, reduction="mean"):
    """Cross entropy of ``softmax(hidden @ weight.T + bias)`` against ``target``, without ever storing the logits.

    ``hidden`` ``[..., D]``, ``weight`` ``[V, D]`` and ``bias`` ``[V]`` are of one type, ``target`` ``[...]`` int64 or int32.
    The loss is float32: per token with ``reduction='none'``, else their sum, or their mean over the tokens that count.
    Tokens whose target is ``ignore_index`` have loss 0 and leave nothing in any gradient, whatever ``hidden`` holds there; if
    no token counts, the loss and its gradients are 0.  A target that is neither ``ignore_index`` nor in ``[0, V)`` gives NaN.
    A bias of ``-inf`` takes a word out."""
    ignore_index, reduction = _decided(ignore_index, reduction)
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _LinearCrossEntropy.apply(hidden, weight, target, bias, ignore_index, reduction)
    device = hidden.device
    with _on(device):
        return _lib.native().cross_entropy(hidden, weight, target, bias, ignore_index, reduction, _stream_of(device))[0]


def linear_cross_entropy_grad(hidden, weight, target, bias=None, ignore_index=-100, reduction="mean"):
    """``(loss, dhidden, dweight, dbias)`` of :func:`linear_cross_entropy` for a gradient of 1 (of ones, with
    ``reduction='none'``), without autograd; ``dbias`` is ``None`` where there is no bias."""
    ignore_index, reduction = _decided(ignore_index, reduction)
    device = hidden.device
    with _on(device):
        return _lib.native().cross_entropy_step(hidden, weight, target, bias, ignore_index, reduction, _stream_of(device))


# ---------------------------------------------------------------------------------------------
# recurrence
# ---------------------------------------------------------------------------------------------

def _recur(x, gate, state, lengths, keep):
    device = x.device
    with _on(device):
        return _lib.native().recurrence(x, gate, state, lengths, keep, _stream_of(device))


class _GatedRecurrence(Function):
    @staticmethod
    def forward(ctx, x, gate, state, lengths):
        out, last, kept = _recur(x, gate, state, lengths, True)
        ctx.save_for_backward(x, gate, lengths, kept)
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, grad_last):
        x, gate, lengths, kept = ctx.saved_tensors
        device, needed = x.device, ctx.needs_input_grad
        if grad is None and grad_last is None:
            return None, None, None, None
        with _on(device):
            dx, dgate, dstate = _lib.native().recurrence_grad(x, gate, grad, grad_last, lengths, kept,
                                                              needed[0] | needed[1] << 1 | needed[2] << 2, _stream_of(device))
        return dx, dgate, dstate, None


def gated_recurrence(x, gate, state=None, lengths=None):
    """``(out, last)`` of the recurrence ``h[t] = a[t] * h[t - 1] + (1 - a[t]) * x[t]`` with ``a = sigmoid(gate)``, channel by
    channel along sequences.

    ``x`` and ``gate`` ``[B, T, D]`` are of one type; they may be pieces of one tensor (``chunk`` of a projection's result).
    ``state`` ``[B, D]`` in float32 is what the sequences begin with, zeros if there is none; ``out`` ``[B, T, D]`` holds every
    ``h``, ``last`` ``[B, D]`` the last ones in float32, to go on from: token by token with ``T`` = 1, or piece by piece.
    ``lengths`` ``[B]`` (int64 or int32, held to ``[0, T]``) ends a sequence early: what ``x`` and ``gate`` hold behind it is not
    looked at, ``out`` and the gradients are 0 there, and ``last`` is the state at its end."""
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or (state is not None and state.requires_grad)):
        return _GatedRecurrence.apply(x, gate, state, lengths)
    return _recur(x, gate, state, lengths, False)[:2]


# ---------------------------------------------------------------------------------------------
# distillation of a linear head
# ---------------------------------------------------------------------------------------------

def _warmth(temperature, reduction):
    """``temperature`` and ``reduction`` as the library takes them."""
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction must be 'none', 'sum' or 'mean', is %r" % (reduction,))
    temperature = float(temperature)
    if not 2.0 ** -20 <= temperature <= 2.0 ** 20:
        raise ValueError("temperature must be from 2^-20 to 2^20, is %r" % temperature)
    return temperature, _REDUCTIONS[reduction]


class _LinearDistillation(Function):
    @staticmethod
    def forward(ctx, hidden, weight, ids, logits, bias, temperature, reduction):
        device = hidden.device
        with _on(device):
            loss, lse, share = _lib.native().distill(hidden, weight, ids, logits, bias, temperature, reduction, _stream_of(device))
        ctx.save_for_backward(hidden, weight, ids, logits, bias, lse, share)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        hidden, weight, ids, logits, bias, lse, share = ctx.saved_tensors
        device, needed = hidden.device, ctx.needs_input_grad
        with _on(device):
            dhidden, dweight, dbias = _lib.native().distill_grad(
                hidden, weight, ids, logits, bias, ctx.temperature, lse, share, grad.float().contiguous(),
                needed[0] | needed[1] << 1 | needed[4] << 2, _stream_of(device))
        return dhidden, dweight, None, None, dbias, None, None


def linear_distillation(hidden, weight, teacher_ids, teacher_logits, bias=None, temperature=1.0, reduction="mean"):
    """How far ``softmax((hidden @ weight.T + bias) / temperature)`` is from a teacher that is known by its best words, without ever
    storing the logits: ``temperature ** 2`` times the Kullback-Leibler divergence of ``q``, the softmax of
    ``teacher_logits / temperature`` over those words.

    ``hidden`` ``[..., D]``, ``weight`` ``[V, D]`` and ``bias`` ``[V]`` are of one type; ``teacher_ids`` ``[..., K]`` (int64 or int32)
    and ``teacher_logits`` ``[..., K]`` (float32, bfloat16 or float16) name 1 to 1024 words for every token, in any order; they get no
    gradient.  A place with a negative number or a logit of ``-inf`` holds none.  A word in two places has both shares, and each
    place its own ``q log q`` in the loss, which is no longer the words' divergence then.  The
    loss is float32: per token with ``reduction='none'``, else their sum, or their mean over the tokens that have a word; tokens
    without one have loss 0 and leave nothing in any gradient.  A number of ``V`` or more, or a logit that is NaN or ``inf``, gives
    NaN."""
    temperature, reduction = _warmth(temperature, reduction)
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _LinearDistillation.apply(hidden, weight, teacher_ids, teacher_logits.detach(), bias, temperature, reduction)
    device = hidden.device
    with _on(device):
        return _lib.native().distill(hidden, weight, teacher_ids, teacher_logits, bias, temperature, reduction, _stream_of(device))[0]


def linear_distillation_grad(hidden, weight, teacher_ids, teacher_logits, bias=None, temperature=1.0, reduction="mean"):
    """``(loss, dhidden, dweight, dbias)`` of :func:`linear_distillation` for a gradient of 1 (of ones, with
    ``reduction='none'``), without autograd; ``dbias`` is ``None`` where there is no bias."""
    temperature, reduction = _warmth(temperature, reduction)
    device = hidden.device
    with _on(device):
        return _lib.native().distill_step(hidden, weight, teacher_ids, teacher_logits, bias, temperature, reduction, _stream_of(device))


# ---------------------------------------------------------------------------------------------
# gated block
# ---------------------------------------------------------------------------------------------

_ACTIVATIONS = {"silu": _lib.DS_SILU, "gelu": _lib.DS_GELU, "relu": _lib.DS_RELU, "sigmoid": _lib.DS_SIGMOID}


def _activation(activation):
    if activation not in _ACTIVATIONS:
        raise ValueError("activation must be 'silu', 'gelu', 'relu' or 'sigmoid', is %r" % (activation,))
    return _ACTIVATIONS[activation]


def _gate(x, weight, bias, activation, keep):
    device = x.device
    with _on(device):
        return _lib.native().gated(x, weight, bias, activation, keep, _stream_of(device))


class _GatedLinear(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation):
        out, halves = _gate(x, weight, bias, activation, True)
        ctx.save_for_backward(x, weight, halves)
        ctx.activation = activation
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, halves = ctx.saved_tensors
        device, needed = x.device, ctx.needs_input_grad
        with _on(device):
            dx, dweight, dbias = _lib.native().gated_grad(x, weight, halves, grad, ctx.activation,
                                                          needed[0] | needed[1] << 1 | needed[2] << 2, _stream_of(device))
        return dx, dweight, dbias, None


def gated_linear(x, weight, bias=None, activation="silu"):
    """``act(x @ gate.T + b) * (x @ up.T + c)``, the gated block of a feed-forward layer, both projections, the activation and the
    product in one kernel: ``weight`` ``[2 F, D]`` is ``gate`` above ``up`` and ``bias`` ``[2 F]`` ``b`` before ``c`` -- what one
    linear layer, or one ``LinearShift``, of ``2 F`` features holds.  ``x`` ``[..., D]``, all of one type; ``activation`` is
    ``'silu'``, ``'gelu'`` (by the error function), ``'relu'`` or ``'sigmoid'``.  For gradients both projections are kept, in
    32 bits; their own gradient is rounded to the type once, for the products that make those of ``x`` and ``weight`` of it."""
    activation = _activation(activation)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _GatedLinear.apply(x, weight, bias, activation)
    return _gate(x, weight, bias, activation, False)[0]


# ---------------------------------------------------------------------------------------------
# clipping
# ---------------------------------------------------------------------------------------------

def _flat(t):
    """Whether the tensor's elements fill one stretch of memory in some order."""
    return t.is_contiguous() or torch.ops.aten.is_non_overlapping_and_dense(t)


def _clip(grads, max_norm, out, scale):
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    outs = None if out is None else [out] if isinstance(out, torch.Tensor) else list(out)
    device = grads[0].device if grads and isinstance(grads[0], torch.Tensor) else torch.device("cpu")
    with _on(device):
        clip = _lib.native().clip
        norm = clip(grads, outs, max_norm, scale, False, _stream_of(device))
        if norm is None:
            # not all contiguous; what is written to copies is copied back, on the same stream
            sources, targets, back = _stretches(grads, grads if outs is None else outs)
            if scale and back:
                _check_apart(grads if outs is None else outs)    # the copies hide what they are copied back to
            norm = clip(sources, None if targets is sources else targets, max_norm, scale, True, _stream_of(device))
            if scale:
                for o, copy in back:
                    o.copy_(copy)
    return norm


def _meet(a, b):
    """Whether two tensors have a byte of memory in common."""
    reach = {}   # by how many bytes an index moves: which differences of indices there are
    for t, other in ((a, False), (b, True)):
        for n, stride in zip(t.shape, t.stride()):
            low, high = reach.get(stride * t.element_size(), (0, 0))
            reach[stride * t.element_size()] = (low - n + 1, high) if other else (low, high + n - 1)
    reach.pop(0, None)
    steps = sorted(((step, low, high) for step, (low, high) in reach.items()), reverse=True)

    def found(steps, least, most):
        """Whether the steps add up to something from ``least`` to ``most``."""
        if not steps:
            return least <= 0 <= most
        (step, low, high), rest = steps[0], steps[1:]
        below, above = sum(s * x for s, x, _ in rest), sum(s * x for s, _, x in rest)
        return any(found(rest, least - x * step, most - x * step)
                   for x in range(max(low, -((above - least) // step)), min(high, (most - below) // step) + 1))

    gap = b.data_ptr() - a.data_ptr()
    return found(steps, gap - a.element_size() + 1, gap + b.element_size() - 1)


def _check_apart(outs):
    """Refuses tensors whose elements are written twice, however they lie in memory."""
    spans = []
    for t in outs:
        if t.numel():
            if any(n > 1 and stride == 0 for n, stride in zip(t.shape, t.stride())):
                raise ValueError("elements of a tensor that is written share their memory")
            length = sum((n - 1) * stride for n, stride in zip(t.shape, t.stride())) + 1
            spans.append((t.data_ptr(), t.data_ptr() + length * t.element_size(), t))
    spans.sort(key=lambda span: span[0])
    open_ = []
    for span in spans:
        open_ = [other for other in open_ if other[1] > span[0]]
        if any(_meet(other[2], span[2]) for other in open_):
            raise ValueError("a tensor is given twice, or one that is written shares memory with another one")
        open_.append(span)


def _stretches(grads, outs):
    """The same calls on tensors whose elements fill stretches of memory in one order, and the results to copy back."""
    sources, targets, back = [], [], []
    for t, o in zip(grads, outs):
        src, dst = t, o
        if t is o:
            if not _flat(t):
                src = dst = t.contiguous()
        elif not (t.is_contiguous() and o.is_contiguous()) and not (t.stride() == o.stride() and _flat(t)):
            src = t.contiguous()
            dst = o if o.is_contiguous() else torch.empty_like(src, dtype=o.dtype)
        if dst is not o:
            back.append((o, dst))
        sources.append(src)
        targets.append(dst)
    return sources, (sources if all([a is b for a, b in zip(sources, targets)]) else targets), back


def gradient_norm(grads):
    """The global 2-norm of all tensors in ``grads``, a float32 scalar on their device."""
    with torch.no_grad():
        return _clip(grads, 0.0, None, False)


def clip_gradients_(grads, max_norm, out=None):
    """Scales ``grads`` by ``min(1, max_norm / (norm + 1e-6))`` and returns ``norm``, their global 2-norm before it (a float32
    scalar on the device; nothing waits for it).  The results go to ``out``, a tensor for each gradient, of any of the three
    types, or in place.  Types may differ from tensor to tensor.  A norm that is infinite or NaN scales by 0 or NaN.  A tensor
    that is written may share no memory with another one, of ``grads`` or of ``out`` (but be its own gradient)."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError("max_norm must not be negative")
    with torch.no_grad():
        return _clip(grads, max_norm, out, True)


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Clips the ``.grad`` of ``parameters`` (those that have one) in place by their global 2-norm, which is returned: the
    counterpart of ``torch.nn.utils.clip_grad_norm_`` for gradients on one device; a ``norm_type`` other than 2 is refused.
    ``error_if_nonfinite`` raises before anything is scaled, and waits for the GPU to know."""
    if isinstance(norm_type, (bool, str)) or norm_type != 2:
        raise ValueError("norm_type must be 2, is %r" % (norm_type,))
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.zeros(())
    if error_if_nonfinite:
        norm = gradient_norm(grads)
        if not torch.isfinite(norm):
            raise RuntimeError("the gradients' norm is %s" % norm.item())
    return clip_gradients_(grads, max_norm)


# ---------------------------------------------------------------------------------------------
# modules
# ---------------------------------------------------------------------------------------------

class ScaledEmbedding(nn.Module):
    """``scale * weight[ids]``; the row of ``padding_idx`` starts at zero and gets no gradient."""

    def __init__(self, num_embeddings, embedding_dim, scale=1.0, padding_idx=None):
        super().__init__()
        self.num_embeddings, self.embedding_dim, self.scale = num_embeddings, embedding_dim, scale
        self.padding_idx = None if padding_idx is None else _padding(padding_idx, num_embeddings)
        self.weight = nn.Parameter(torch.empty(num_embeddings, embedding_dim))
        self.reset_parameters()

    def reset_parameters(self):
        nn.init.normal_(self.weight, std=1.0 / self.scale if self.scale else 1.0)
        if self.padding_idx is not None:
            with torch.no_grad():
                self.weight[self.padding_idx].zero_()

    def forward(self, ids):
        return embedding(ids, self.weight, self.scale, self.padding_idx)

    def extra_repr(self):
        return "{num_embeddings}, {embedding_dim}, scale={scale}, padding_idx={padding_idx}".format(**self.__dict__)


class LinearCrossEntropy(nn.Module):
    """A linear head and its cross entropy in one module: ``forward(hidden, target)`` is the loss, :meth:`logits` what an
    ``nn.Linear`` of the same weight would give."""

    def __init__(self, in_features, num_classes, bias=True, ignore_index=-100, reduction="mean"):
        super().__init__()
        if reduction not in _REDUCTIONS:
            raise ValueError("reduction must be 'none', 'sum' or 'mean', is %r" % (reduction,))
        self.in_features, self.num_classes = in_features, num_classes
        self.ignore_index, self.reduction = ignore_index, reduction
        head = nn.Linear(in_features, num_classes, bias=bias)
        self.weight, self.bias = head.weight, head.bias

    def forward(self, hidden, target):
        return linear_cross_entropy(hidden, self.weight, target, self.bias, self.ignore_index, self.reduction)

    def distill(self, hidden, teacher_ids, teacher_logits, temperature=1.0):
        """:func:`linear_distillation` of this head, reduced as its loss is."""
        return linear_distillation(hidden, self.weight, teacher_ids, teacher_logits, self.bias, temperature, self.reduction)

    def logits(self, hidden):
        return nn.functional.linear(hidden, self.weight, self.bias)

    def extra_repr(self):
        return "{}, {}, bias={}, ignore_index={}, reduction={}".format(
            self.in_features, self.num_classes, self.bias is not None, self.ignore_index, self.reduction)


class GatedLinear(nn.Module):
    """:func:`gated_linear` with a weight and a bias of its own, drawn as an ``nn.Linear`` of ``2 * out_features`` draws them."""

    def __init__(self, in_features, out_features, bias=True, activation="silu"):
        super().__init__()
        _activation(activation)
        self.in_features, self.out_features, self.activation = in_features, out_features, activation
        both = nn.Linear(in_features, 2 * out_features, bias=bias)
        self.weight, self.bias = both.weight, both.bias

    def forward(self, x):
        return gated_linear(x, self.weight, self.bias, self.activation)

    def extra_repr(self):
        return "{}, {}, bias={}, activation={!r}".format(self.in_features, self.out_features, self.bias is not None, self.activation)


class GatedShift(nn.Module):
    """The gated block with weights of powers of two: ``layer`` is one ``LinearShift`` (``shift_type`` ``'PS'``) or ``LinearShiftQ``
    (``'Q'``) of twice the width, whose float path's weights go into :func:`gated_linear`; straight-through gradients reach its
    parameters.  With ``use_kernel`` (no gradients) the layer runs on the shift kernels, and the gate behind it.  A ``layer`` that
    is there already is taken as it is."""

    def __init__(self, in_features, out_features, bias=True, activation="silu", shift_type="PS", layer=None, **options):
        super().__init__()
        if shift_type not in ("PS", "Q"):
            raise ValueError("shift_type must be 'PS' or 'Q', is %r" % (shift_type,))
        _activation(activation)
        self.in_features, self.out_features, self.activation = in_features, out_features, activation
        if layer is None:
            kind = modules.LinearShift if shift_type == "PS" else modules_q.LinearShiftQ
            layer = kind(in_features, 2 * out_features, bias=bias, **options)
        elif (layer.in_features, layer.out_features) != (in_features, 2 * out_features):
            raise ValueError("layer must have %d features and give %d, has %d and gives %d" % (
                in_features, 2 * out_features, layer.in_features, layer.out_features))
        self.layer = layer

    def forward(self, x):
        layer = self.layer
        if layer.use_kernel:
            gate, up = layer(x).chunk(2, -1)
            return getattr(nn.functional if self.activation in ("silu", "gelu") else torch, self.activation)(gate) * up
        return gated_linear(layer.float_input(x), layer.float_weight(), layer.bias, self.activation)

    def extra_repr(self):
        return "{}, {}, activation={!r}".format(self.in_features, self.out_features, self.activation)
