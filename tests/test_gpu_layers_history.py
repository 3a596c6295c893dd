"""What linear and gated_linear remember of a call: second derivatives are refused wherever there would be one, and nothing else is; what is
kept for the backward pass is what the gradients that can be asked for read."""
import itertools

import pytest
import torch

import lmms_engine_amd as E

pytestmark = pytest.mark.gpu
DEV = "cuda"
ACTS = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu}
NAMES = {"linear": ("x", "w", "b", "r"), "gated": ("x", "wg", "wu", "bg", "bu")}


def inputs(kind, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(5)
    t, k, n = 6, 16, 8
    shape = dict(x=(t, k), w=(n, k), wg=(n, k), wu=(n, k), b=(n,), bg=(n,), bu=(n,), r=(t, n))
    return {m: (torch.randn(*shape[m], generator=g, device=DEV) * 0.5).to(dtype) for m in NAMES[kind]}


def call(kind, v, act):
    if kind == "linear":
        return E.linear(v["x"], v["w"], v["b"], activation=act, residual=v["r"])
    return E.gated_linear(v["x"], v["wg"], v["wu"], v["bg"], v["bu"], activation=act)


def plain(kind, v, act):
    f = ACTS[act]
    if kind == "linear":
        return f(v["x"] @ v["w"].t() + v["b"]) + v["r"]
    return f(v["x"] @ v["wg"].t() + v["bg"]) * (v["x"] @ v["wu"].t() + v["bu"])


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("kind", list(NAMES))
def test_no_second_derivative_is_dropped(kind, act):
    """One or two inputs are trained, the gradient of one of them goes into a loss beside another term, and the loss is differentiated by each.
    Where the plain form has a second derivative the call raises, by .backward() and by autograd.grad alike; where it has none the loss's
    gradient is the other term's."""
    base = inputs(kind)
    for trained in itertools.chain(itertools.combinations(base, 1), itertools.combinations(base, 2)):
        for asked, by in itertools.product(trained, trained):
            wide = {m: a.double().requires_grad_(m in trained) for m, a in base.items()}
            (first,) = torch.autograd.grad(plain(kind, wide, act).sum(), wide[asked], create_graph=True)
            second = torch.autograd.grad(first.square().sum(), wide[by], allow_unused=True)[0] if first.requires_grad else None
            there = second is not None and bool(second.any())
            for whole in (False, True):
                v = {m: a.clone().requires_grad_(m in trained) for m, a in base.items()}
                (first,) = torch.autograd.grad(call(kind, v, act).sum(), v[asked], create_graph=True)
                loss = first.square().sum() + v[by].square().sum()
                case = (trained, asked, by, whole)
                # .backward() runs through everything that the loss depends on, by whichever input
                reached = there if not whole else first.requires_grad
                if reached:
                    with pytest.raises(RuntimeError, match="differentiated once"):
                        loss.backward() if whole else torch.autograd.grad(loss, v[by])
                    assert there or whole, case
                    continue
                assert not there, case
                if whole:
                    loss.backward()
                    got = v[by].grad
                else:
                    (got,) = torch.autograd.grad(loss, v[by])
                assert torch.equal(got, 2 * base[by]), case


@pytest.mark.parametrize("kind", list(NAMES))
def test_a_gradient_has_a_history_where_the_plain_form_has_one(kind):
    """For every pair of inputs and activations without a kink: requires_grad of a gradient is that of the formula's."""
    base = inputs(kind)
    for act in ("none", "silu"):
        for trained in itertools.chain(itertools.combinations(base, 1), itertools.combinations(base, 2)):
            got, want = ({m: a.clone().requires_grad_(m in trained) for m, a in base.items()} for _ in range(2))
            leaves = [m for m in base if m in trained]
            first = torch.autograd.grad(call(kind, got, act).sum(), [got[m] for m in leaves], create_graph=True)
            plainly = torch.autograd.grad(plain(kind, want, act).sum(), [want[m] for m in leaves], create_graph=True)
            for m, a, e in zip(leaves, first, plainly):
                assert a.requires_grad == e.requires_grad, (act, trained, m)


@pytest.mark.parametrize("kind", list(NAMES))
def test_a_loss_whose_gradient_has_a_history_closes_every_gradient(kind):
    """The incoming gradient depends on the inputs: so does every gradient, whichever input is trained."""
    base = inputs(kind)
    for act, asked in itertools.product(ACTS, base):
        v = {m: a.clone().requires_grad_(m == asked) for m, a in base.items()}
        (first,) = torch.autograd.grad(call(kind, v, act).square().sum(), v[asked], create_graph=True)
        assert first.requires_grad
        if asked == "r":  # the incoming gradient itself
            (second,) = torch.autograd.grad(first.sum(), v["r"])
            assert torch.equal(second, torch.full_like(second, 2.0))
            continue
        with pytest.raises(RuntimeError, match="differentiated once"):
            torch.autograd.grad(first.square().sum() + v[asked].square().sum(), v[asked])


def grads_of(kind, base, trained, act, between):
    """Gradients by `trained` of a call between whose passes `between` is done with its inputs."""
    v = {m: a.clone().requires_grad_(m in trained) for m, a in base.items()}
    used = {m: a * 1 if m in trained else a for m, a in v.items()}  # (a leaf that is trained cannot be changed in place)
    y = call(kind, used, act)
    between(used)
    return dict(zip(trained, torch.autograd.grad(y, [v[m] for m in trained], torch.ones_like(y))))


# what the gradient by an input reads beside what is kept of the activation
READS = {"linear": dict(x="w", w="x", b="", r=""), "gated": dict(x=("wg", "wu"), wg="x", wu="x", bg="", bu="")}


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("kind", list(NAMES))
def test_inputs_that_no_gradient_reads_may_change(kind, act):
    """An input that is changed in place between the passes: the gradients that do not read it are what they were, those that do raise."""
    base = inputs(kind)
    for trained in itertools.chain(itertools.combinations(base, 1), itertools.combinations(base, 2)):
        want = grads_of(kind, base, trained, act, lambda v: None)
        for changed in base:
            def change(v):
                with torch.no_grad():
                    v[changed].mul_(3).add_(1)

            if any(changed in READS[kind][m] for m in trained):
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    grads_of(kind, base, trained, act, change)
                continue
            got = grads_of(kind, base, trained, act, change)
            for m in trained:
                assert torch.equal(got[m], want[m]), (trained, changed, m)


@pytest.mark.parametrize("dtype,each", [(torch.bfloat16, 3), (torch.float32, 4)], ids=["bf16", "f32"])
def test_what_is_kept_is_what_is_read(dtype, each):
    """Memory between the passes, beside the result: the factors that the gradients need and no input that they do not."""
    t, k, n = 1024, 2048, 512  # buffers of whole megabytes each
    mb = 1 << 20

    def kept(f, **shapes):
        """Bytes that the call holds on to once the caller has let go of what it passed."""
        asked = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]  # (allocated ones count what is left of a cached block too)
        before = asked()
        v = {m: torch.zeros(*s, dtype=dtype, device=DEV) for m, s in shapes.items()}
        y = f(v)
        del v
        return asked() - before - y.numel() * y.element_size()

    factor, size = t * n * each, torch.finfo(dtype).bits // 8
    x, w, b = t * k * size, n * k * size, n * size
    slack = 64 * 1024
    shapes = dict(x=(t, k), w=(n, k), w2=(n, k), b=(n,), b2=(n,), r=(t, n))

    def trained(*names, **call):
        def f(v):
            for m in names:
                v[m].requires_grad_(True)
            if "w2" in v:
                return E.gated_linear(v["x"], v["w"], v["w2"], v["b"], v["b2"], **call)
            return E.linear(v["x"], v["w"], v["b"], residual=v["r"], **call)
        return f

    def pick(*names):
        return {m: shapes[m] for m in names}

    lin, gated = pick("x", "w", "b", "r"), pick("x", "w", "w2", "b", "b2")
    # (a trained leaf lives on in its own gradient's node)
    for names, act, want in ((("x",), "none", x + w), (("w",), "none", x + w), (("b",), "none", b), (("r",), "silu", t * n * size),
                             (("b",), "silu", b + factor), (("x",), "silu", x + w + factor)):
        got = kept(trained(*names, activation=act), **lin)
        assert abs(got - want) <= slack, (names, act, got / mb, want / mb)
    for names, want in ((("b",), b + factor), (("b2",), b + factor), (("w",), w + x + factor), (("w2",), w + x + factor), (("x",), x + 2 * w + 2 * factor),
                        (("b", "b2"), 2 * b + 2 * factor)):
        got = kept(trained(*names), **gated)
        assert abs(got - want) <= slack, (names, got / mb, want / mb)


@pytest.mark.parametrize("which", ["x", "w", "b", "r"])
def test_a_tensor_whose_memory_was_freed_is_refused(which):
    """Sharded training frees a parameter's storage and keeps the tensor: it is not taken for one that was left out."""
    v = inputs("linear")
    v[which].untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="freed"):
        call("linear", v, "silu")
    if which != "r":
        with pytest.raises(ValueError, match="freed"):
            E.gated_linear(v["x"], v["w"], v["w"], v["b"], v["b"])
