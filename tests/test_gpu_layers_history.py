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
