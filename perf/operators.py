"""The operators at the two ends of a token model's training step, and on its gradients, as measurable cases: the
scaled embedding lookup and its gradient, the cross entropy of a linear head over a large vocabulary with its gradients,
and the clipping of gradients by their global norm.

``listed()`` names the standing cases, ``draw(rng)`` gives others of the same ranges; ``prepare`` builds what a program
holds before the call, ``run`` makes one pass (the plain form in 32 bits, or the package's operators where ``own`` is
true), ``work`` counts what the pass cannot do without and ``exact`` computes the same results in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_IGNORE = -100

# What real programs keep per tensor: the parameters of the networks that this package converts, and stacks of square
# layers with their two vectors.
_SETS = ("mlp", "resnet18", "resnet50", "stack")


def _embed(T, V, D, dtype, scale=1.0):
    return dict(kind="embed", T=T, V=V, D=D, dtype=dtype, scale=scale)


def _embed_grad(T, V, D, dtype, scale=1.0, padded=0.0):
    return dict(kind="embed_grad", T=T, V=V, D=D, dtype=dtype, scale=scale, padded=padded)


def _loss(T, D, V, dtype, bias, ignored=0.0, step=True, shift=False):
    return dict(kind="loss", T=T, D=D, V=V, dtype=dtype, bias=bias, ignored=ignored, step=step, shift=shift)


def _clip(tensors, dtype, count=1, width=0, active=True):
    return dict(kind="clip", tensors=tensors, dtype=dtype, count=count, width=width, active=active)


def listed():
    named = [
        # 64 tokens, one of each sequence of a served batch: nothing but latency
        ("embed_b64", _embed(64, 1000, 512, "f32", math.sqrt(512))),
        # the lookup of a whole training batch from a table of 1 GB
        ("embed_b131072", _embed(131072, 131072, 4096, "bf16", 64.0)),
        # a ragged batch of a small model, a third of it padding: one row collects 700 gradients
        ("embed_grad_odd", _embed_grad(2065, 10007, 385, "f32", math.sqrt(385), 0.34)),
        # the gradient of a large table for a large batch: most of it is rows of zeros
        ("embed_grad_b65536", _embed_grad(65536, 131072, 2048, "bf16", 1.0, 0.0)),
        # the classifier of a ResNet-18 whose weights are powers of two, batch 64: latency
        ("loss_resnet18_b64", _loss(64, 512, 1000, "f32", True, shift=True)),
        # scoring of a few candidate tokens, no gradient: bound by reading the head's weights
        ("loss_score_37", _loss(37, 2048, 50021, "bf16", False, step=False)),
        # odd in every dimension, a fifth of the tokens not counted
        ("loss_f16_odd", _loss(1543, 1000, 20011, "f16", True, 0.2)),
        # float32 training, the type of this package's modules
        ("loss_f32_b2048", _loss(2048, 1024, 32768, "f32", True)),
        # a large step: 8192 tokens over 131072 words
        ("loss_bf16_b8192", _loss(8192, 4096, 131072, "bf16", False, 0.05)),
        # gradients of the MNIST MLP, six small tensors: latency
        ("clip_mlp", _clip("mlp", "f32")),
        # gradients of a ResNet-50, 161 tensors of all sizes, in place, with a norm that needs no clipping
        ("clip_resnet50_inactive", _clip("resnet50", "f32", active=False)),
        # bfloat16 gradients of a deep stack into the float32 buffers of an optimizer: 0.8 G elements
        ("clip_stack_bf16", _clip("stack", "bf16", 48, 4096)),
    ]
    return [dict(case, name=name) for name, case in named]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "embed_grad", "loss", "loss", "clip"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind in ("embed", "embed_grad"):
        V = _log_int(rng, 100, 131072)
        D = _log_int(rng, 32, 4096)
        if rng.random() < 0.5:
            D = max(64, D // 64 * 64)
        scale = rng.choice([1.0, math.sqrt(D)])
        if kind == "embed":
            return _embed(_log_int(rng, 1, 65536), V, D, dtype, scale)
        return _embed_grad(_log_int(rng, 1, 32768), V, D, dtype, scale, rng.choice([0.0, 0.3, 0.9]))
    if kind == "loss":
        T, D, V = _log_int(rng, 1, 8192), _log_int(rng, 64, 4096), _log_int(rng, 10, 131072)
        if rng.random() < 0.5:
            D = max(64, D // 64 * 64)
        budget = 2e12 if dtype == "f32" else 4e12
        while T * D * V > budget:
            T = max(1, T // 2)
        return _loss(T, D, V, dtype, rng.random() < 0.5, rng.choice([0.0, 0.0, 0.3]), step=rng.random() < 0.7,
                     shift=rng.random() < 0.3)
    tensors = rng.choice(_SETS)
    return _clip(tensors, dtype, rng.randint(1, 48) if tensors == "stack" else 1,
                 _log_int(rng, 33, 2048) if tensors == "stack" else 0, rng.random() < 0.7)


def _shapes(case):
    """The shapes of the gradients a program of this kind clips."""
    tensors = case["tensors"]
    if tensors == "mlp":
        sizes = (784, 512, 512, 10)
        return [s for a, b in zip(sizes[:-1], sizes[1:]) for s in ((b, a), (b,))]
    if tensors == "stack":
        w = case["width"]
        return [s for _ in range(case["count"]) for s in ((w, w), (w,), (w,))]
    shapes = [(64, 3, 7, 7), (64,), (64,)]
    cin = 64
    for i, depth in enumerate((2, 2, 2, 2) if tensors == "resnet18" else (3, 4, 6, 3)):
        w = 64 * 2 ** i
        for j in range(depth):
            if tensors == "resnet18":
                convs, cout = [(w, cin, 3, 3), (w, w, 3, 3)], w
            else:
                convs, cout = [(w, cin, 1, 1), (w, w, 3, 3), (4 * w, w, 1, 1)], 4 * w
            if j == 0 and (i > 0 or cin != cout):
                convs.append((cout, cin, 1, 1))
            for c in convs:
                shapes += [c, (c[0],), (c[0],)]
            cin = cout
    return shapes + [(1000, cin), (1000,)]


def _flat(case, dtype, dev):
    """One buffer, and the gradients as pieces of it that begin at multiples of 64 elements."""
    shapes = _shapes(case)
    starts = [0]
    for s in shapes:
        starts.append(starts[-1] + -(-math.prod(s) // 64) * 64)
    flat = torch.zeros(starts[-1], dtype=dtype, device=dev)
    return flat, [flat[at:at + math.prod(s)].view(s) for at, s in zip(starts, shapes)]


def _tokens(T, V, g, dev):
    """Token numbers as text has them: the k-th most frequent one with a frequency near 1/k, numbered at random."""
    rank = torch.rand(T, generator=g, device=dev, dtype=torch.float64).mul_(math.log(V + 1)).exp_().floor_().long() - 1
    return torch.randperm(V, generator=g, device=dev)[rank.clamp_(0, V - 1)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    kind = case["kind"]
    if kind == "clip":
        flat, grads = _flat(case, _TYPES[case["dtype"]], dev)
        for i, t in enumerate(grads):
            t.copy_(torch.randn(t.shape, generator=g, device=dev) * (0.02 * 4.0 ** (i % 3 - 1)))
        # an active clip goes to the optimizer's float32 buffers, one that finds nothing to do works in place
        whole, out = _flat(case, torch.float32, dev) if case["active"] else (flat, None)
        return dict(case=case, grads=grads, out=out, whole=whole, max_norm=1.0 if case["active"] else 1e6)
    dtype = _TYPES[case["dtype"]]
    T, V, D = case["T"], case["V"], case["D"]
    ids = _tokens(T, V, g, dev)
    if kind == "embed":
        weight = (torch.randn(V, D, generator=g, device=dev) * 0.02).to(dtype)
        return dict(case=case, ids=ids, weight=weight)
    if kind == "embed_grad":
        # padding (token 0) fills the ends of the sequences; its row gets no gradient when it is named as padding, and
        # collects all of them here
        ids[T - int(T * case["padded"]):] = 0
        grad = (torch.randn(T, D, generator=g, device=dev) * 1e-2).to(dtype)
        return dict(case=case, ids=ids, grad=grad)
    hidden = torch.randn(T, D, generator=g, device=dev).to(dtype)
    if case["shift"]:
        # a head of powers of two, as a shift layer of five bits holds them (scaled for logits of ordinary size)
        w = 2.0 ** torch.randint(-14, 1, (V, D), generator=g, device=dev).float()
        w *= torch.randint(0, 2, (V, D), generator=g, device=dev) * 2 - 1
        w *= 2.0 ** -round(math.log2(math.sqrt(D) / 7))
    else:
        w = torch.randn(V, D, generator=g, device=dev) * (2.0 / math.sqrt(D))
    weight = w.to(dtype)
    bias = (torch.randn(V, generator=g, device=dev) * 0.1).to(dtype) if case["bias"] else None
    ids[torch.rand(T, generator=g, device=dev) < case["ignored"]] = _IGNORE
    return dict(case=case, hidden=hidden, weight=weight, bias=bias, target=ids)


def _run_own(state):
    from deepshift_amd import training
    case = state["case"]
    if case["kind"] == "embed":
        return training.embedding(state["ids"], state["weight"], scale=case["scale"])
    if case["kind"] == "embed_grad":
        return training.embedding_grad(state["ids"], state["grad"], case["V"], scale=case["scale"])
    if case["kind"] == "loss":
        args = (state["hidden"], state["weight"], state["target"], state["bias"])
        if not case["step"]:
            return training.linear_cross_entropy(*args, ignore_index=_IGNORE, reduction="none")
        return _named(training.linear_cross_entropy_grad(*args, ignore_index=_IGNORE, reduction="mean"))
    return dict(norm=training.clip_gradients_(state["grads"], state["max_norm"], out=state["out"]), grads=state["whole"])


def _named(results):
    loss, dhidden, dweight, dbias = results
    named = dict(loss=loss, dhidden=dhidden, dweight=dweight)
    if dbias is not None:
        named["dbias"] = dbias
    return named


def run(state):
    with torch.no_grad():
        if own:
            return _run_own(state)
        case = state["case"]
        if case["kind"] == "embed":
            weight = state["weight"]
            return (weight[state["ids"]].float() * case["scale"]).to(weight.dtype)
        if case["kind"] == "embed_grad":
            grad = state["grad"]
            total = torch.zeros(case["V"], case["D"], device=grad.device)
            total.index_add_(0, state["ids"], grad.float())
            return (total * case["scale"]).to(grad.dtype)
        if case["kind"] == "clip":
            return _plain_clip(state)
        return _plain_loss(state)


def _plain_loss(state):
    hidden, weight, bias, target = state["hidden"], state["weight"], state["bias"], state["target"]
    h, w = hidden.float(), weight.float()
    logits = h @ w.t()
    if bias is not None:
        logits += bias.float()
    top = logits.amax(1, keepdim=True)
    logsum = top[:, 0] + (logits - top).exp_().sum(1).log_()
    counted = target != _IGNORE
    at = target.clamp(min=0)[:, None]
    losses = torch.where(counted, logsum - logits.gather(1, at)[:, 0], 0.0)
    if not state["case"]["step"]:
        return losses
    share = counted.float() / counted.sum().clamp(min=1)
    p = logits.sub_(logsum[:, None]).exp_()
    p.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float32))
    p *= share[:, None]
    dbias = None if bias is None else p.sum(0).to(bias.dtype)
    return _named(((losses * share).sum(), (p @ w).to(hidden.dtype), (p.t() @ h).to(weight.dtype), dbias))


def _plain_clip(state):
    grads, out = state["grads"], state["out"]
    norm = torch.stack([t.float().square().sum() for t in grads]).sum().sqrt()
    factor = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    for i, t in enumerate(grads):
        (t if out is None else out[i]).copy_(t.float() * factor)
    return dict(norm=norm, grads=state["whole"])


def work(case):
    kind, b = case["kind"], _SIZE[case["dtype"]]
    if kind == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        # read for the norm; the result is written, from what was read, where the norm asks for it
        return {"bytes": n * (b + (4 if case["active"] else 0)), "flops": n * (3 if case["active"] else 2)}
    T, V, D = case["T"], case["V"], case["D"]
    if kind == "embed":
        # the rows that T draws are expected to reach, once each, and the result
        k = torch.arange(1, V + 1, dtype=torch.float64)
        reached = int((1.0 - (1.0 - torch.log1p(1.0 / k) / math.log(V + 1)) ** T).sum())
        return {"bytes": T * 8 + (reached + T) * D * b, "flops": T * D}
    if kind == "embed_grad":
        return {"bytes": T * 8 + (T + V) * D * b, "flops": T * D}
    product = 2 * T * D * V
    size = (T * D + V * D + (V if case["bias"] else 0)) * b + T * 8
    if not case["step"]:
        return {"bytes": size + T * 4, "flops": product}
    return {"bytes": 2 * size, "flops": 3 * product}


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind == "embed":
            T, D = case["T"], case["D"]
            out = torch.empty(T, D, dtype=torch.float64, device="cuda")
            for i in range(0, T, 8192):
                out[i:i + 8192] = torch.index_select(state["weight"], 0, state["ids"][i:i + 8192]).double()
            return out.mul_(case["scale"])
        if kind == "embed_grad":
            order = torch.argsort(state["ids"], stable=True)
            sums = torch.zeros(case["V"], case["D"], dtype=torch.float64, device="cuda")
            for part in order.split(8192):
                sums.index_add_(0, state["ids"][part], state["grad"][part].double(), alpha=case["scale"])
            return sums
        if kind == "clip":
            norm = math.sqrt(sum(torch.linalg.vector_norm(t.double()).item() ** 2 for t in state["grads"]))
            factor = min(1.0, state["max_norm"] / (norm + 1e-6))
            whole, parts = _flat(case, torch.float64, "cuda")
            for part, t in zip(parts, state["grads"]):
                part.copy_(t).mul_(factor)
            return dict(norm=torch.tensor(norm, dtype=torch.float64, device="cuda"), grads=whole)
        return _exact_loss(case, state)


def _exact_loss(case, state):
    """Blocks of tokens, each with its whole row of logits in 64 bits."""
    T, D, V = case["T"], case["D"], case["V"]
    w = state["weight"].double()
    b = state["bias"].double() if case["bias"] else None
    target = state["target"]
    kept = (target != _IGNORE)
    n = max(1, int(kept.sum()))
    losses = torch.zeros(T, dtype=torch.float64, device="cuda")
    if case["step"]:
        dh = torch.zeros(T, D, dtype=torch.float64, device="cuda")
        dw = torch.zeros(V, D, dtype=torch.float64, device="cuda")
        db = torch.zeros(V, dtype=torch.float64, device="cuda")
    block = max(1, min(T, 2 ** 29 // V))
    for i in range(0, T, block):
        rows = slice(i, min(T, i + block))
        h = state["hidden"][rows].double()
        z = torch.mm(h, w.t())
        if b is not None:
            z = z + b
        logp = torch.log_softmax(z, dim=1)
        keep, where = kept[rows], target[rows].clamp(min=0)
        picked = logp[torch.arange(len(where), device="cuda"), where]
        losses[rows] = torch.where(keep, -picked, torch.zeros_like(picked))
        if case["step"]:
            e = logp.exp()
            e[torch.arange(len(where), device="cuda"), where] -= 1.0
            e *= (keep.double() / n)[:, None]
            dh[rows] = torch.mm(e, w)
            dw += torch.mm(e.t(), h)
            db += e.sum(0)
    if not case["step"]:
        return losses
    return _named((losses.sum() / n, dh, dw, db if case["bias"] else None))
