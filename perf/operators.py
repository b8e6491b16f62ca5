"""Performance cases of the operators of a decoder's training step, on one GPU.

* ``ce``      ``linear_cross_entropy``: the head's product and the softmax cross entropy over the vocabulary, with the gradients of the
  hidden states and of the head's weight (``grad``), or the loss alone, as an evaluation asks for it;
* ``norm``    ``residual_norm``: a block's output goes through its norm, gate and residual scale into the residual stream, and the
  stream through the next block's norm; forward and backward;
* ``swiglu``  ``swiglu8``: the gated activation of an MLP, whose inputs are kept in 8 bits and used in the backward pass;
* ``pack``    ``pack8`` and ``unpack8``: a block's input kept in 8 bits, and what the recomputation gets back.

``own`` false: the plain form, elementary operations in 32 bits.  ``own`` true: the package's operators.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORED = -100
GROUP = 64              # features that share one scale where activations are kept in 8 bits
EPS = 1e-5
LARGEST = 8192 * 4096 * 128256


def listed():
    return [
        # the tiny preset's head, eight sequences of sixteen tokens: launches and host time
        dict(name="ce_128x32x64", kind="ce", tokens=128, hidden=32, vocab=64, dtype="bf16", reduction="mean", grad=True, ignored=0.0),
        # one rank's eighth of a 128256-word head on one sequence
        dict(name="ce_4096x4096x16032", kind="ce", tokens=4096, hidden=4096, vocab=16032, dtype="bf16", reduction="mean", grad=True, ignored=0.0),
        # the whole head on two sequences
        dict(name="ce_8192x4096x128256", kind="ce", tokens=8192, hidden=4096, vocab=128256, dtype="bf16", reduction="mean", grad=True, ignored=0.0),
        # ragged in every direction, a quarter of the tokens padding, weighted token by token by the caller
        dict(name="ce_1999x1000x32003", kind="ce", tokens=1999, hidden=1000, vocab=32003, dtype="fp16", reduction="none", grad=True, ignored=0.25),
        # evaluation of a few prompts: the loss of each token, no gradients
        dict(name="ce_eval_515x2048x50021", kind="ce", tokens=515, hidden=2048, vocab=50021, dtype="bf16", reduction="none", grad=False, ignored=0.1),
        # the tiny preset's norm
        dict(name="norm_128x32", kind="norm", rows=128, dim=32, dtype="bf16", after=False, gate=False, scale=1.0),
        # one sequence of hidden size 4096: the residual sum and the next norm
        dict(name="norm_4096x4096", kind="norm", rows=4096, dim=4096, dtype="bf16", after=False, gate=False, scale=1.0),
        # four sequences with a norm after the block, a gate and a residual scale
        dict(name="norm_16384x4096_gated", kind="norm", rows=16384, dim=4096, dtype="bf16", after=True, gate=True, scale=0.5),
        # one rank's eighth of an MLP of 14336, a ragged batch
        dict(name="swiglu_4097x1792", kind="swiglu", rows=4097, dim=1792, dtype="bf16"),
        # the whole MLP on two sequences
        dict(name="swiglu_8192x14336", kind="swiglu", rows=8192, dim=14336, dtype="bf16"),
        # a block's input: the tiny preset's, and eight sequences of hidden size 4096
        dict(name="pack_128x32", kind="pack", rows=128, dim=32, dtype="bf16"),
        dict(name="pack_32768x4096", kind="pack", rows=32768, dim=4096, dtype="bf16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))


def _width(rng, low, high):
    """Mostly a multiple of 64, as widths are; sometimes any number."""
    value = _spread(rng, low, high)
    return value if value < 64 or rng.random() < 0.35 else value // 64 * 64


def draw(rng):
    kind = rng.choice(("ce", "ce", "norm", "norm", "swiglu", "pack"))
    if kind == "ce":
        hidden, vocab = _width(rng, 32, 4096), _spread(rng, 64, 128256)
        tokens = _spread(rng, 1, 8192)
        return dict(kind=kind, tokens=tokens, hidden=hidden, vocab=vocab, dtype=rng.choice(("bf16", "bf16", "fp16")),
                    reduction=rng.choice(("mean", "sum", "none")), grad=rng.random() < 0.75, ignored=rng.choice((0.0, 0.1, 0.4)))
    if kind == "norm":
        dim = _width(rng, 32, 8192)
        rows = _spread(rng, 1, min(32768, 16384 * 4096 // dim))
        return dict(kind=kind, rows=rows, dim=dim, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), after=rng.random() < 0.5,
                    gate=rng.random() < 0.5, scale=rng.choice((1.0, 0.5, 0.1767767)))
    dim = _width(rng, 32, 14336)
    return dict(kind=kind, rows=_spread(rng, 1, min(32768, 8192 * 14336 // dim)), dim=dim, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")))


def work(case):
    """Bytes: inputs once, outputs once, and what the backward pass needs of the forward one kept (written and read once)."""
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "ce":
        n, d, v = case["tokens"], case["hidden"], case["vocab"]
        per_token = n if case["reduction"] == "none" else 1
        moved = size * (n * d + v * d) + 8 * n + 4 * per_token
        if case["grad"]:
            moved += size * (n * d + v * d) + (4 * n if case["reduction"] == "none" else 0)
        return {"bytes": moved, "flops": (6 if case["grad"] else 2) * n * d * v}
    n = case["rows"] * case["dim"]
    if case["kind"] == "norm":
        # x, branch, gh, gy in; h, y, dx and the branch's gradient out (dx again where nothing lies between them); both kept and read again
        streams = 4 + 2 + (2 if case["after"] or case["gate"] or case["scale"] != 1.0 else 1) + 1 + (1 if case["after"] or case["gate"] else 0)
        vectors = 2 * (1 + case["after"] + case["gate"])
        return {"bytes": size * (n * streams + vectors * case["dim"]), "flops": 20 * n}
    kept = n + 4 * case["rows"] * -(-case["dim"] // GROUP)
    if case["kind"] == "swiglu":
        return {"bytes": size * 6 * n + 4 * kept, "flops": 40 * n}
    return {"bytes": size * 2 * n + 2 * kept, "flops": 4 * n}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _stream(g, rows, dim):
    """A residual stream or a block's output: tokens of different size, a few features far larger than the others."""
    features = torch.where(torch.rand(dim, generator=g, device="cuda") < 0.01, 8.0, 1.0)
    return _normal(g, rows, dim) * features * torch.exp(0.5 * _normal(g, rows, 1))


def prepare(case, seed):
    g = _generator(seed)
    dtype = TYPES[case["dtype"]]
    state = {"case": dict(case)}
    if case["kind"] == "ce":
        n, d, v = case["tokens"], case["hidden"], case["vocab"]
        weight = _normal(g, v, d).mul_(1.25 / math.sqrt(d)).to(dtype)
        targets = torch.randint(0, v, (n,), generator=g, device="cuda")
        # normed hidden states that have learnt something: the right word's logit is raised by 0 to 16, token by token
        known = 16.0 * torch.rand(n, 1, generator=g, device="cuda")
        hidden = (_normal(g, n, d) + known / 1.5625 * weight[targets].float()).to(dtype)
        # padding at the end of the batch, and single tokens inside it that do not count
        padded = int(0.8 * case["ignored"] * n)
        targets[n - padded:] = IGNORED
        targets[torch.rand(n, generator=g, device="cuda") < 0.2 * case["ignored"]] = IGNORED
        state |= {"hidden": hidden, "weight": weight, "targets": targets}
        if case["reduction"] == "none":
            state["grad_loss"] = torch.rand(n, generator=g, device="cuda") + 0.5
        leaves = ("hidden", "weight") if case["grad"] else ()
    elif case["kind"] == "norm":
        n, d = case["rows"], case["dim"]
        state |= {"x": _stream(g, n, d).to(dtype), "branch": (0.5 * _stream(g, n, d)).to(dtype), "weight": (1 + 0.1 * _normal(g, d)).to(dtype),
                  "grad_h": _normal(g, n, d).to(dtype), "grad_y": _normal(g, n, d).to(dtype)}
        if case["after"]:
            state["branch_weight"] = (1 + 0.1 * _normal(g, d)).to(dtype)
        if case["gate"]:
            state["gate"] = (0.5 + 0.2 * _normal(g, d)).to(dtype)
        leaves = ("x", "branch", "weight") + (("branch_weight",) if case["after"] else ()) + (("gate",) if case["gate"] else ())
    elif case["kind"] == "swiglu":
        n, d = case["rows"], case["dim"]
        state |= {"gate": _stream(g, n, d).to(dtype), "up": _stream(g, n, d).to(dtype), "grad_y": _normal(g, n, d).to(dtype)}
        leaves = ("gate", "up")
    else:
        state["x"] = _stream(g, case["rows"], case["dim"]).to(dtype)
        leaves = ()
    for name in leaves:
        state[name].requires_grad_()
    state["leaves"] = leaves
    return state


# ---------------------------------------------------------------------------------------------------------------------
# The package's operators, as a program calls them.
def _own(state):
    from soap_tp_b200 import ops

    case = state["case"]
    leaves = [state[name] for name in state["leaves"]]
    if case["kind"] == "ce":
        loss = ops.linear_cross_entropy(state["hidden"], state["weight"], state["targets"], reduction=case["reduction"], ignore_index=IGNORED)
        if not case["grad"]:
            return {"loss": loss}
        grads = torch.autograd.grad(loss, leaves, state.get("grad_loss"))
        return {"loss": loss.detach(), "grads": grads}
    if case["kind"] == "norm":
        h, y = ops.residual_norm(state["x"], state["branch"], state["weight"], branch_weight=state.get("branch_weight"),
                                 gate=state.get("gate"), scale=case["scale"], eps=EPS)
        grads = torch.autograd.grad((h, y), leaves, (state["grad_h"], state["grad_y"]))
        return {"h": h.detach(), "y": y.detach(), "grads": grads}
    if case["kind"] == "swiglu":
        y = ops.swiglu8(state["gate"], state["up"])
        return {"y": y.detach(), "grads": torch.autograd.grad(y, leaves, state["grad_y"])}
    return {"x": ops.unpack8(ops.pack8(state["x"]))}


# ---------------------------------------------------------------------------------------------------------------------
# The plain form.
def _plain_ce(state):
    case = state["case"]
    hidden, weight, targets = state["hidden"].detach(), state["weight"].detach(), state["targets"]
    h, w = hidden.float(), weight.float()
    counted = targets != IGNORED
    at = torch.where(counted, targets, 0).unsqueeze(1)
    logits = h @ w.t()
    most = logits.max(dim=1, keepdim=True).values
    picked = logits.gather(1, at) - most
    exp = logits.sub_(most).exp_()
    total = exp.sum(dim=1, keepdim=True)
    losses = torch.where(counted, (total.log() - picked).squeeze(1), 0.0)
    number = counted.sum().clamp(min=1).float()
    loss = losses if case["reduction"] == "none" else losses.sum() if case["reduction"] == "sum" else losses.sum() / number
    if not case["grad"]:
        return {"loss": loss}
    factor = state["grad_loss"] if case["reduction"] == "none" else torch.ones_like(losses) if case["reduction"] == "sum" else (1.0 / number).expand_as(losses)
    factor = torch.where(counted, factor, 0.0).unsqueeze(1)
    d = exp.div_(total).mul_(factor)
    d.scatter_add_(1, at, -factor)
    return {"loss": loss, "grads": ((d @ w).to(hidden.dtype), (d.t() @ h).to(weight.dtype))}


def _plain_norm(state):
    case = state["case"]
    dtype = state["x"].dtype
    x, b, w = (state[k].detach().float() for k in ("x", "branch", "weight"))
    one = torch.ones_like(w)
    gate = state["gate"].detach().float() if case["gate"] else one
    if case["after"]:
        wb = state["branch_weight"].detach().float()
        rb = 1.0 / (b.square().mean(dim=1, keepdim=True) + EPS).sqrt()
        n = b * rb * wb
    else:
        n = b
    h = x + case["scale"] * gate * n
    r = 1.0 / (h.square().mean(dim=1, keepdim=True) + EPS).sqrt()
    y = h * r * w
    gy = state["grad_y"].float()
    t = gy * w
    dh = state["grad_h"].float() + r * (t - h * (r * r) * (t * h).mean(dim=1, keepdim=True))
    dn = case["scale"] * gate * dh
    grads = [dh, dn, (gy * h * r).sum(dim=0)]
    if case["after"]:
        t = dn * wb
        grads[1] = rb * (t - b * (rb * rb) * (t * b).mean(dim=1, keepdim=True))
        grads.append((dn * b * rb).sum(dim=0))
    if case["gate"]:
        grads.append((case["scale"] * dh * n).sum(dim=0))
    return {"h": h.to(dtype), "y": y.to(dtype), "grads": [v.to(dtype) for v in grads]}


def _plain_kept(x):
    """The values that 8 bits and one scale for GROUP features hold of x, in 32 bits."""
    rows, dim = x.shape
    groups = -(-dim // GROUP)
    v = torch.nn.functional.pad(x.detach().float(), (0, groups * GROUP - dim)).view(rows, groups, GROUP)
    scale = (v.abs().amax(dim=2, keepdim=True) / 127.0).clamp(min=2.0 ** -126)
    return (torch.round(v / scale) * scale).view(rows, groups * GROUP)[:, :dim]


def _plain_swiglu(state):
    dtype = state["gate"].dtype
    g, u, dy = state["gate"].detach().float(), state["up"].detach().float(), state["grad_y"].float()
    y = g / (1.0 + (-g).exp()) * u
    g, u = _plain_kept(state["gate"]), _plain_kept(state["up"])
    s = 1.0 / (1.0 + (-g).exp())
    return {"y": y.to(dtype), "grads": ((dy * u * s * (1.0 + g * (1.0 - s))).to(dtype), (dy * g * s).to(dtype))}


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "ce":
        return _plain_ce(state)
    if kind == "norm":
        return _plain_norm(state)
    if kind == "swiglu":
        return _plain_swiglu(state)
    return {"x": _plain_kept(state["x"]).to(state["x"].dtype)}


# ---------------------------------------------------------------------------------------------------------------------
# From the definitions, in 64 bits.
def _exact_ce(case, state):
    w = state["weight"].detach().double()
    targets = state["targets"]
    n = targets.numel()
    counted = targets != IGNORED
    number = max(1, int(counted.sum()))
    losses = torch.zeros(n, dtype=torch.float64, device="cuda")
    d_hidden = torch.zeros(n, w.shape[1], dtype=torch.float64, device="cuda") if case["grad"] else None
    d_weight = torch.zeros_like(w) if case["grad"] else None
    for start in range(0, n, 2048):
        h = state["hidden"].detach()[start:start + 2048].double()
        t, mine = targets[start:start + 2048], counted[start:start + 2048]
        log_p = torch.log_softmax(h @ w.t(), dim=1)
        right = torch.zeros_like(log_p)
        index = mine.nonzero().squeeze(1)
        right[index, t[index]] = 1.0
        losses[start:start + 2048] = -(log_p * right).sum(dim=1)
        if case["grad"]:
            per = {"none": state.get("grad_loss", losses)[start:start + 2048].double(), "sum": torch.ones_like(losses[start:start + 2048]),
                   "mean": torch.full_like(losses[start:start + 2048], 1.0 / number)}[case["reduction"]]
            d = (log_p.exp_() - right) * (per * mine).unsqueeze(1)
            d_hidden[start:start + 2048] = d @ w
            d_weight += d.t() @ h
    loss = {"none": losses, "sum": losses.sum(), "mean": losses.sum() / number}[case["reduction"]]
    return {"loss": loss, "grads": (d_hidden, d_weight)} if case["grad"] else {"loss": loss}


def _exact_norm(case, state):
    names = list(state["leaves"])
    v = {k: state[k].detach().double().requires_grad_() for k in names}

    def norm(z):
        return z * torch.rsqrt(z.pow(2).mean(dim=-1, keepdim=True) + EPS)

    b = v["branch"]
    if case["after"]:
        b = norm(b) * v["branch_weight"]
    if case["gate"]:
        b = b * v["gate"]
    h = v["x"] + b * case["scale"]
    y = norm(h) * v["weight"]
    grads = torch.autograd.grad((h, y), [v[k] for k in names], (state["grad_h"].double(), state["grad_y"].double()))
    return {"h": h.detach(), "y": y.detach(), "grads": list(grads)}


def _exact_kept(x):
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    for start in range(0, x.shape[1], GROUP):
        part = x[:, start:start + GROUP].detach().double()
        step = (part.abs().max(dim=1, keepdim=True).values / 127).clamp_min(2.0 ** -126)
        out[:, start:start + GROUP] = (part / step).round() * step
    return out


def _exact_swiglu(state):
    y = torch.nn.functional.silu(state["gate"].detach().double()) * state["up"].detach().double()
    g, u = _exact_kept(state["gate"]).requires_grad_(), _exact_kept(state["up"]).requires_grad_()
    grads = torch.autograd.grad(g * torch.sigmoid(g) * u, (g, u), state["grad_y"].double())
    return {"y": y, "grads": grads}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "ce":
        return _exact_ce(case, state)
    if case["kind"] == "norm":
        return _exact_norm(case, state)
    if case["kind"] == "swiglu":
        return _exact_swiglu(state)
    return {"x": _exact_kept(state["x"])}
