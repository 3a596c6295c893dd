"""The operators that stand around the products of a model's layers, row by row, as cases that can be timed.

  embedding   `embedding`: rows of a table times a scale, and the table's gradient
  layer_norm  `layer_norm`: (s - mean) / sqrt(var + eps) * weight + bias of s = x + residual, and its gradients
  rms_norm    `rms_norm`: s / sqrt(mean(s^2) + eps) * weight, and its gradients
  dropout     `dropout`: residual + x / (1 - p) where a counter-based generator keeps x, and its gradient from the same numbers

`listed()` holds the calls of a model's life, from one token that is being answered to a training step over a long sequence; `draw()` gives
more of the same ranges.  Where `own` is false, `run` computes the formulas with elementary torch operations in 32 bits; where it is true, it
calls the framework.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "bf16": 2}
DEFAULTS = dict(train=True, dtype="bf16")
EMBEDDING = dict(DEFAULTS, kind="embedding", scaled=False, share=0.0)
NORM = dict(DEFAULTS, residual=True)
LAYER_NORM = dict(NORM, kind="layer_norm", eps=1e-5)
RMS_NORM = dict(NORM, kind="rms_norm", eps=1e-6)
DROPOUT = dict(DEFAULTS, kind="dropout", p=0.1, residual=True, site=0)


def listed():
    return [
        # the last token of an answer is looked up: latency is all
        dict(EMBEDDING, name="embedding_token", tokens=1, inner=4096, vocab=151936, train=False),
        # a training step over a long sequence with a large table, a third of it placeholders of image patches: one id thousands of times
        dict(EMBEDDING, name="embedding_train", tokens=8192, inner=4096, vocab=151936, share=0.33),
        # a small model in single precision, sizes that are no multiple of anything, scaled by the root of its width
        dict(EMBEDDING, name="embedding_train_odd", tokens=1777, inner=251, vocab=10007, dtype="f32", scaled=True),
        # a batch of answers, one token each, between two blocks
        dict(LAYER_NORM, name="layer_norm_tokens", rows=24, inner=1024, train=False),
        # a block of an image encoder in training
        dict(LAYER_NORM, name="layer_norm_train_encoder", rows=4096, inner=1024),
        # single precision on odd features, without a residual
        dict(LAYER_NORM, name="layer_norm_train_odd", rows=777, inner=251, dtype="f32", residual=False),
        # one token of one answer between two blocks
        dict(RMS_NORM, name="rms_norm_token", rows=1, inner=4096, train=False),
        # between two blocks in training, over a long sequence: the residual stream is read, added to and written
        dict(RMS_NORM, name="rms_norm_train", rows=8192, inner=4096),
        # the heads of queries, each normalised by itself: many short rows
        dict(RMS_NORM, name="rms_norm_train_heads", rows=8192 * 32, inner=128, residual=False),
        # behind the attention of a small model, with the residual
        dict(DROPOUT, name="dropout_train_small", rows=512, inner=896, site=3),
        # behind the activation of a large feed-forward block, over a long sequence
        dict(DROPOUT, name="dropout_train", rows=8192, inner=12288, residual=False, site=17),
        # an odd number of values in single precision
        dict(DROPOUT, name="dropout_train_odd", rows=1237, inner=333, dtype="f32", p=0.25, site=1),
    ]


def most(kind):
    return max(work(c)["bytes"] for c in listed() if c["kind"] == kind)


def draw(rng):
    def size(low, high, whole=1):
        n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        return max(whole, n // whole * whole)

    kind = rng.choice(("embedding", "layer_norm", "rms_norm", "dropout"))
    common = dict(train=rng.random() < 0.7, dtype="f32" if rng.random() < 0.3 else "bf16")
    # three widths in four are whole cache lines, as model sizes are; the others are anything
    inner = size(64, 12288, 64 if rng.random() < 0.75 else 1)
    if kind == "embedding":
        # (a share of a half and more of one id is a prompt of pictures)
        case = dict(EMBEDDING, **{**common, "scaled": rng.random() < 0.3, "share": rng.choice((0.0, 0.0, 0.2, 0.6))}, tokens=size(1, 32768),
                    inner=min(inner, 8192), vocab=size(512, 160000))
    elif kind == "dropout":
        case = dict(DROPOUT, **{**common, "residual": rng.random() < 0.6, "p": rng.choice((0.05, 0.1, 0.2, 0.5, rng.random())), "site": rng.randrange(100)},
                    rows=size(1, 16384), inner=inner)
    else:
        case = dict(LAYER_NORM if kind == "layer_norm" else RMS_NORM, **{**common, "residual": rng.random() < 0.6}, rows=size(1, 16384), inner=inner)
        if rng.random() < 0.2:  # heads
            case.update(rows=size(64, 262144), inner=rng.choice((64, 80, 128, 256)))
    while work(case)["bytes"] > most(kind):
        longer = "rows" if kind != "embedding" else "vocab" if case["vocab"] > case["tokens"] else "tokens"
        case[longer] //= 2
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, train, kind = DTYPES[case["dtype"]], case["train"], case["kind"]
    n = case["inner"]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale

    def leaf(v):
        return v.to(dt).requires_grad_(train)

    def gradient(*shape):  # of a run under way: rows differ in size
        return (normal(*shape, scale=1e-3) * torch.exp(normal(shape[0], 1, scale=0.7))).to(dt) if train else None

    if kind == "embedding":
        t, v = case["tokens"], case["vocab"]
        # words by rank: the k-th most frequent one about 1 / k of the time, and the placeholders in one piece
        ids = torch.exp(torch.rand(t, generator=g, device="cuda", dtype=torch.float64) * math.log(v)).long().clamp_(1, v) - 1
        first, some = t // 5, int(t * case["share"])
        ids[first:first + some] = v - 3
        return dict(case=case, ids=ids, weight=leaf(normal(v, n, scale=0.02)), scale=math.sqrt(n) if case["scaled"] else 1.0, dy=gradient(t, n))
    rows = case["rows"]
    # activations, some features of which are larger than the others; a residual stream that earlier blocks have added to
    x = leaf(normal(rows, n) * torch.exp(normal(n, scale=0.5)) + (0.2 if kind == "layer_norm" else 0.0))
    residual = leaf(normal(rows, n, scale=3.0) + normal(n)) if case["residual"] else None
    state = dict(case=case, x=x, residual=residual, dy=gradient(rows, n))
    if kind == "dropout":
        state["seed"] = (seed * 0x9E3779B97F4A7C15 + 0x1234567) % 2 ** 64
        return state
    state["weight"] = leaf(1.0 + normal(n, scale=0.3))
    state["bias"] = leaf(normal(n, scale=0.1)) if kind == "layer_norm" else None
    state["ds"] = gradient(rows, n) if case["residual"] else None  # what comes back along the residual stream
    return state


def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return PLAIN[case["kind"]](state, DTYPES[case["dtype"]])
    from lmms_engine_amd import dropout, embedding, layer_norm, rms_norm

    kind, train = case["kind"], case["train"]
    if kind == "embedding":
        y = embedding(state["ids"], state["weight"], scale=state["scale"])
        if not train:
            return {"y": y}
        (dw,) = torch.autograd.grad(y, [state["weight"]], state["dy"])
        return {"y": y.detach(), "dweight": dw}
    x, residual = state["x"], state["residual"]
    if kind == "dropout":
        y = dropout(x, case["p"], seed=state["seed"], site=case["site"], residual=residual)
        outs, incoming = [y], [state["dy"]]
    elif kind == "layer_norm":
        y = layer_norm(x, state["weight"], state["bias"], eps=case["eps"], residual=residual)
    else:
        y = rms_norm(x, state["weight"], eps=case["eps"], residual=residual)
    out = {}
    if kind != "dropout":
        outs, incoming = (list(y), [state["dy"], state["ds"]]) if residual is not None else ([y], [state["dy"]])
        if residual is not None:
            out["s"] = outs[1].detach()
    out["y"] = outs[0].detach()
    if train:
        named = leaves(state)
        out.update({"d" + name: g for name, g in zip(named, torch.autograd.grad(outs, list(named.values()), incoming))})
    return out


def leaves(state):
    """What a training step differentiates by."""
    return {name: state[name] for name in ("x", "residual", "weight", "bias") if state.get(name) is not None}


# ---- the formulas in 32 bits ----------------------------------------------------------------------


def plain_embedding(state, dt):
    ids, scale = state["ids"], state["scale"]
    out = {"y": (state["weight"][ids].float() * scale).to(dt)}
    if state["dy"] is not None:
        dw = torch.zeros(state["weight"].shape, device=ids.device)
        dw.index_add_(0, ids, state["dy"].float())
        out["dweight"] = (dw * scale).to(dt)
    return out


def plain_norm(state, dt):
    case = state["case"]
    centred = case["kind"] == "layer_norm"
    s, w, out = state["x"], state["weight"].float(), {}
    if case["residual"]:
        s = out["s"] = (s.float() + state["residual"].float()).to(dt)  # the stream that goes on, which is what is normalised
    s = s.float()
    if centred:
        s = s - s.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((s * s).mean(1, keepdim=True) + case["eps"])
    hat = s * rstd
    y = hat * w
    out["y"] = (y + state["bias"].float() if centred else y).to(dt)
    if not case["train"]:
        return out
    dy = state["dy"].float()
    g = dy * w
    dx = g - hat * (g * hat).mean(1, keepdim=True)
    if centred:
        dx = dx - g.mean(1, keepdim=True)
        out["dbias"] = dy.sum(0).to(dt)
    dx = dx * rstd
    if case["residual"]:
        dx = dx + state["ds"].float()
        out["dresidual"] = dx.to(dt)
    out["dx"] = dx.to(dt)
    out["dweight"] = (dy * hat).sum(0).to(dt)
    return out


def philox(c, key):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers, as easy as 1, 2, 3; 2011) of four words of counters."""
    mask = 0xFFFFFFFF
    k0, k1 = key & mask, key >> 32
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # (the 64 bits of each product, whatever their sign says)
        c = [(b >> 32 & mask) ^ c[1] ^ k0, b & mask, (a >> 32 & mask) ^ c[3] ^ k1, a & mask]
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return c


def uniform(count, key, site, device):
    """The 32-bit number of each value of a tensor: the upper halves of eight values are a block of the generator, their lower halves another."""
    group = torch.arange(-(-count // 8), device=device)
    halves = []
    for which in (0, 1):
        words = philox([group & 0xFFFFFFFF, group >> 32, torch.full_like(group, site), torch.full_like(group, which)], key)
        halves.append(torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], dim=1).reshape(-1)[:count])
    return halves[0] << 16 | halves[1]


def plain_dropout(state, dt):
    case, x = state["case"], state["x"].float()
    limit = round(case["p"] * 2 ** 32)
    keep = (uniform(x.numel(), state["seed"], case["site"], x.device) >= limit).view(x.shape)
    scale = 2 ** 32 / (2 ** 32 - limit)
    zero = torch.zeros((), device=x.device)
    y = torch.where(keep, x * scale, zero)
    if case["residual"]:
        y = y + state["residual"].float()
    out = {"y": y.to(dt)}
    if case["train"]:
        out["dx"] = torch.where(keep, state["dy"].float() * scale, zero).to(dt)
        if case["residual"]:
            out["dresidual"] = state["dy"].clone()
    return out


PLAIN = {"embedding": plain_embedding, "layer_norm": plain_norm, "rms_norm": plain_norm, "dropout": plain_dropout}


def work(case):
    size, train, n = SIZES[case["dtype"]], case["train"], case["inner"]
    if case["kind"] == "embedding":
        t, v = case["tokens"], case["vocab"]
        values = (min(t, v) + t) * n + ((t + v) * n if train else 0)
        return {"bytes": values * size + 8 * t, "flops": t * n * (2 if train else 1)}
    rows = case["rows"]
    # x and the residual are read, y (and of a norm the sum) is written; dy (and ds) is read, dx is written, to the residual goes dy or dx itself
    streams = 2 + case["residual"] * (1 if case["kind"] == "dropout" else 2)
    if train:
        streams += 2 + (case["residual"] if case["kind"] != "dropout" else 0)
    values = streams * rows * n
    if case["kind"] == "dropout":
        return {"bytes": values * size, "flops": rows * n * (30 if train else 15)}
    values += (2 if case["kind"] == "layer_norm" else 1) * n * (2 if train else 1)
    return {"bytes": values * size, "flops": rows * n * (20 if train else 8)}


# ---- the definitions in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    """The definitions once more in 64 bits, gradients by autograd's rules."""
    state = prepare(case, seed)
    train, kind = case["train"], case["kind"]
    if kind == "embedding":
        table = state["weight"].detach().double()
        out = {"y": torch.index_select(table, 0, state["ids"]) * state["scale"]}
        if train:
            del table
            out["dweight"] = torch.zeros(state["weight"].shape, dtype=torch.float64, device="cuda").index_add_(
                0, state["ids"], state["dy"].double() * state["scale"])
        return out
    wide = {name: v.detach().double().requires_grad_(train) for name, v in leaves(state).items()}
    if kind == "dropout":
        limit = round(case["p"] * 2 ** 32)
        kept = (numbers(wide["x"].numel(), state["seed"], case["site"]) >= limit).view_as(wide["x"])
        y = torch.where(kept, wide["x"] / (1 - limit / 2 ** 32), 0.0)
        outs = [y + wide["residual"] if case["residual"] else y]
        out, incoming = {"y": outs[0].detach()}, [state["dy"]]
    else:
        s, out = wide["x"], {}
        outs, incoming = [], [state["dy"]]
        if case["residual"]:
            s = s + wide["residual"]
            out["s"] = s.detach()
            outs, incoming = [s], [state["ds"], state["dy"]]
            s = s + (s.detach().to(DTYPES[case["dtype"]]).double() - s.detach())  # what goes on is held in the tensors' type
        if kind == "layer_norm":
            y = torch.nn.functional.layer_norm(s, s.shape[-1:], wide["weight"], wide["bias"], case["eps"])
        else:
            y = wide["weight"] * s * torch.rsqrt(s.square().mean(-1, keepdim=True) + case["eps"])
        out["y"] = y.detach()
        outs.append(y)
    if train:
        grads = torch.autograd.grad(outs, list(wide.values()), [v.double() for v in incoming])
        out.update({"d" + name: g for name, g in zip(wide, grads)})
    return out


def numbers(count, key, site):
    """The generator again, its products put together from halves."""
    def wide(m, c):
        low, high = (m & 0xFFFF) * c, (m >> 16) * c
        high = high + (low >> 16)
        return high >> 16, (high & 0xFFFF) << 16 | (low & 0xFFFF)

    at = torch.arange(count, device="cuda")
    block = torch.arange((count + 7) // 8, device="cuda")
    result = torch.zeros_like(at)
    for half in range(2):
        x = torch.stack([block % 2 ** 32, block // 2 ** 32, torch.full_like(block, site), torch.full_like(block, half)])
        for r in range(10):
            ka, kb = ((key % 2 ** 32) + r * 0x9E3779B9) % 2 ** 32, ((key // 2 ** 32) + r * 0xBB67AE85) % 2 ** 32
            (h0, l0), (h1, l1) = wide(0xD2511F53, x[0]), wide(0xCD9E8D57, x[2])
            x = torch.stack([h1 ^ x[1] ^ ka, l1, h0 ^ x[3] ^ kb, l0])
        part = x[(at % 8) // 2, at // 8] >> (16 * (at % 2)) & 0xFFFF
        result = result * 2 ** 16 + part
    return result
