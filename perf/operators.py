"""The layer operators of this framework as cases that can be timed: the products whose weights `Muon` trains.

  linear  `linear`: act(x W^T + bias) + residual, alone or with its backward pass
  gated   `gated_linear`: act(x Wg^T + bg) * (x Wu^T + bu), alone or with its backward pass

`listed()` holds the calls of a model's life, from one token of a small batch that is being answered to a training step over a long
sequence; `draw()` gives more of the same ranges.  Where `own` is false, `run` computes the formulas with elementary torch operations in 32
bits; where it is true, it calls the framework.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "bf16": 2}
ACTIVATIONS = ("none", "relu", "sigmoid", "silu", "gelu", "gelu_tanh")
LARGEST = 3 * 2 * 8192 * 4096 * 2 * 12288  # floating point operations of the largest listed case
LARGEST_F32 = LARGEST // 64
DEFAULTS = dict(bias=False, residual=False, activation="none", train=False, dtype="bf16")


def listed():
    return [
        # one token of one answer goes through the attention's output projection: the weight is read once, latency is all
        dict(DEFAULTS, name="linear_token", kind="linear", tokens=1, inner=4096, outer=4096, residual=True),
        # a batch of answers, one token each, through the down projection of the feed-forward block
        dict(DEFAULTS, name="linear_batch_of_tokens", kind="linear", tokens=24, inner=12288, outer=4096, residual=True),
        # the first layer of an encoder's feed-forward block in training: bias and activation
        dict(DEFAULTS, name="linear_train_encoder", kind="linear", tokens=4096, inner=1024, outer=4096, bias=True, activation="relu", train=True),
        # the down projection of a large block in training, residual included
        dict(DEFAULTS, name="linear_train_down", kind="linear", tokens=8192, inner=12288, outer=4096, residual=True, train=True),
        # sizes of which none is a multiple of anything: a head over an odd number of classes on odd features
        dict(DEFAULTS, name="linear_train_odd", kind="linear", tokens=777, inner=251, outer=1001, bias=True, residual=True, activation="silu", train=True),
        # a small model that is trained in single precision
        dict(DEFAULTS, name="linear_train_f32", kind="linear", tokens=2048, inner=1408, outer=512, bias=True, residual=True, activation="gelu_tanh", train=True,
             dtype="f32"),
        # one token through the gate and up projections of a large block
        dict(DEFAULTS, name="gated_token", kind="gated", tokens=1, inner=4096, outer=12288, activation="silu"),
        # a batch of tokens through those of a small block
        dict(DEFAULTS, name="gated_batch_of_tokens", kind="gated", tokens=53, inner=896, outer=4864, activation="silu"),
        # a prompt of ordinary length, its last rows no whole tile
        dict(DEFAULTS, name="gated_prompt", kind="gated", tokens=1900, inner=4096, outer=12288, activation="silu"),
        # a training step over a long sequence: the largest
        dict(DEFAULTS, name="gated_train", kind="gated", tokens=8192, inner=4096, outer=12288, activation="silu", train=True),
        # the tokens that a router has sent to one expert
        dict(DEFAULTS, name="gated_train_expert", kind="gated", tokens=517, inner=2048, outer=768, activation="silu", train=True),
        # a small model in single precision, with biases
        dict(DEFAULTS, name="gated_train_f32", kind="gated", tokens=1024, inner=512, outer=1408, bias=True, activation="gelu", train=True, dtype="f32"),
    ]


def draw(rng):
    def size(low, high, whole):
        n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        return max(whole, n // whole * whole)

    kind = rng.choice(("linear", "gated"))
    case = dict(DEFAULTS, kind=kind, train=rng.random() < 0.5, dtype="f32" if rng.random() < 0.2 else "bf16", bias=rng.random() < 0.4,
                residual=kind == "linear" and rng.random() < 0.5, activation=rng.choice(ACTIVATIONS if kind == "linear" else ACTIVATIONS[1:]))
    if case["dtype"] == "f32" and case["train"] and case["activation"] == "relu":
        # the gradient jumps where a sum is zero, and at single precision a sum in another order may lie on the other side of it
        case["activation"] = "silu"
    # three features in four are whole cache lines, as model sizes are; the others are anything
    whole = 64 if rng.random() < 0.75 else 1
    case.update(tokens=size(1, 8192, 1), inner=size(64, 12288, whole), outer=size(64, 12288, whole))
    most = LARGEST_F32 if case["dtype"] == "f32" else LARGEST
    while work(case)["flops"] > most:
        case["tokens"] = max(1, case["tokens"] // 2)
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, train = DTYPES[case["dtype"]], case["train"]
    t, k, n = case["tokens"], case["inner"], case["outer"]

    def normal(*shape, scale):
        return torch.randn(*shape, generator=g, device="cuda") * scale

    def leaf(v):
        return v.to(dt).requires_grad_(train)

    # activations behind a norm, some features of which are larger than the others; weights and gradients of a run under way
    x = leaf(normal(t, k, scale=1.0) * torch.exp(normal(k, scale=0.5)))
    weights = [leaf(normal(n, k, scale=0.7 / math.sqrt(k))) for _ in range(2 if case["kind"] == "gated" else 1)]
    biases = [leaf(normal(n, scale=0.1)) if case["bias"] else None for _ in weights]
    residual = leaf(normal(t, n, scale=1.0)) if case["residual"] else None
    dy = (normal(t, n, scale=1e-3) * torch.exp(normal(t, 1, scale=0.7))).to(dt) if train else None
    return dict(case=case, x=x, weights=weights, biases=biases, residual=residual, dy=dy)


def run(state):
    case = state["case"]
    if own:
        from lmms_engine_amd import gated_linear, linear

        x, weights, biases, residual = state["x"], state["weights"], state["biases"], state["residual"]
        if case["kind"] == "linear":
            y = linear(x, weights[0], biases[0], activation=case["activation"], residual=residual)
        else:
            y = gated_linear(x, weights[0], weights[1], biases[0], biases[1], activation=case["activation"])
        if not case["train"]:
            return {"y": y}
        named = leaves(state)
        grads = torch.autograd.grad(y, list(named.values()), state["dy"])
        return {"y": y.detach(), **{"d" + name: g for name, g in zip(named, grads)}}
    with torch.no_grad():
        return plain(state, DTYPES[case["dtype"]])


def leaves(state):
    """What a training step differentiates by, in the order of the outputs."""
    named = {"x": state["x"]}
    named.update({"w%d" % i: w for i, w in enumerate(state["weights"])})
    named.update({"b%d" % i: b for i, b in enumerate(state["biases"]) if b is not None})
    if state["residual"] is not None:
        named["residual"] = state["residual"]
    return named


def activate(name, z):
    """(act(z), act'(z))"""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.clamp(z, min=0), (z > 0).to(z.dtype)
    if name == "gelu":
        phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + th), 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * (c * (1 + 3 * 0.044715 * z * z))
    s = 1 / (1 + torch.exp(-z))
    return (s, s * (1 - s)) if name == "sigmoid" else (z * s, s * (1 + z * (1 - s)))


def plain(state, dt):
    case = state["case"]
    x, weights = state["x"].float(), [w.float() for w in state["weights"]]
    z = [x @ w.t() if b is None else x @ w.t() + b.float() for w, b in zip(weights, state["biases"])]
    a, da = activate(case["activation"], z[0])
    y = a * z[1] if case["kind"] == "gated" else a
    if state["residual"] is not None:
        y = y + state["residual"].float()
    out = {"y": y.to(dt)}
    if not case["train"]:
        return out
    dy = state["dy"].float()
    dz = [dy * z[1] * da, dy * a] if case["kind"] == "gated" else [dy * da]
    dx = dz[0] @ weights[0] if len(dz) == 1 else dz[0] @ weights[0] + dz[1] @ weights[1]
    out["dx"] = dx.to(dt)
    out.update({"dw%d" % i: (d.t() @ x).to(dt) for i, d in enumerate(dz)})
    if case["bias"]:
        out.update({"db%d" % i: d.sum(0).to(dt) for i, d in enumerate(dz)})
    if state["residual"] is not None:
        out["dresidual"] = state["dy"].clone()
    return out


def work(case):
    t, k, n, size = case["tokens"], case["inner"], case["outer"], SIZES[case["dtype"]]
    pair = 2 if case["kind"] == "gated" else 1
    one = t * k + pair * n * k + t * n + (pair * n if case["bias"] else 0) + (t * n if case["residual"] else 0)
    flops = 2 * t * k * n * pair
    if not case["train"]:
        return {"bytes": one * size, "flops": flops}
    # forward and backward: x, the weights, the residual and dy are read, y and every gradient are written
    grads = t * k + pair * n * k + (pair * n if case["bias"] else 0) + (t * n if case["residual"] else 0)
    return {"bytes": (one + t * n + grads) * size, "flops": 3 * flops}


def exact(case, seed):
    """The definition once more in 64 bits: the product by autograd's own rules, over torch's reference functions."""
    import torch.nn.functional as F

    functions = {"none": lambda v: v, "relu": F.relu, "sigmoid": torch.sigmoid, "silu": F.silu, "gelu": F.gelu,
                 "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}
    state = prepare(case, seed)
    wide = {name: v.detach().double().requires_grad_(case["train"]) for name, v in leaves(state).items()}
    hidden = F.linear(wide["x"], wide["w0"], wide.get("b0"))
    y = functions[case["activation"]](hidden)
    if case["kind"] == "gated":
        y = y * F.linear(wide["x"], wide["w1"], wide.get("b1"))
    if "residual" in wide:
        y = y + wide["residual"]
    out = {"y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad(y, list(wide.values()), state["dy"].double())
        out.update({"d" + name: g for name, g in zip(wide, grads)})
    return out
