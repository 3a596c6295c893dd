"""What linear and gated_linear keep for their backward pass, when it is not there any more, or not what it was."""
import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks

import lmms_engine_amd as E

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16]
SHAPES = {"linear": dict(x=(6, 16), w=(8, 16), b=(8,)), "gated": dict(x=(6, 16), wg=(8, 16), wu=(8, 16), bg=(8,), bu=(8,))}


def part(values):
    """The values behind others of their memory: what is left of their address once that is freed is not null."""
    return torch.cat([values.flatten()[:1].expand(16), values.flatten()])[16:].view(values.shape)


def inputs(kind, dtype):
    g = torch.Generator(device=DEV).manual_seed(5)
    return {m: part((torch.randn(shape, generator=g, device=DEV) * 0.5).to(dtype)).requires_grad_(True) for m, shape in SHAPES[kind].items()}


def call(kind, v):
    if kind == "linear":
        return E.linear(v["x"], v["w"], v["b"], activation="silu")
    return E.gated_linear(v["x"], v["wg"], v["wu"], v["bg"], v["bu"])


def free(t):
    t.untyped_storage().resize_(0)


# what each input's gradient reads of the others
READS = {"linear": {"x": ["w"], "w": ["x"], "b": []}, "gated": {"x": ["wg", "wu"], "wg": ["x"], "wu": ["x"], "bg": [], "bu": []}}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,asked", [(k, a) for k in READS for a in READS[k]])
def test_memory_that_was_freed_is_refused_where_it_is_read(kind, asked, dtype):
    """A version counter does not tell that it is gone."""
    for gone in READS[kind]:
        v = inputs(kind, dtype)
        y = call(kind, v)
        dy = torch.ones_like(y)
        (want,) = torch.autograd.grad(y, v[asked], dy, retain_graph=True)
        free(v[gone])
        if gone in READS[kind][asked]:
            with pytest.raises(ValueError, match="freed"):
                torch.autograd.grad(y, v[asked], dy)
        else:
            assert torch.equal(torch.autograd.grad(y, v[asked], dy)[0], want)


@pytest.mark.parametrize("kind", list(SHAPES))
def test_an_incoming_gradient_that_was_freed(kind):
    v = inputs(kind, torch.float32)
    y = call(kind, v)
    dy = part(torch.ones_like(y))
    free(dy)
    with pytest.raises(ValueError, match="freed"):
        torch.autograd.grad(y, list(v.values()), dy)


OTHERS = {
    "a type": (lambda t: t.to(torch.float16 if t.is_floating_point() else torch.int8), TypeError),
    "a wider type": (lambda t: t.double(), TypeError),
    "a device": (lambda t: t.cpu(), ValueError),
    "fewer values": (lambda t: t.flatten()[:0], ValueError),
    "fewer columns": (lambda t: t[..., :-1], ValueError),
    "a shape": (lambda t: torch.stack([t, t]), ValueError),
    "a layout": (lambda t: t.to_sparse(), NotImplementedError),
}


@pytest.mark.parametrize("other", list(OTHERS))
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", list(SHAPES))
def test_what_hooks_give_back_is_what_was_kept(kind, dtype, other):
    change, error = OTHERS[other]
    count = {"linear": 3, "gated": 5}[kind]
    for i in range(count):
        seen, v = [], inputs(kind, dtype)
        with saved_tensors_hooks(lambda t: seen.append(t) or (len(seen) - 1, t), lambda p: change(p[1]) if p[0] == i else p[1]):
            y = call(kind, v)
        assert len(seen) == count
        with pytest.raises(error, match="kept for a backward pass"):
            torch.autograd.grad(y, list(v.values()), torch.ones_like(y))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", list(SHAPES))
def test_hooks_may_give_back_other_strides_and_addresses(kind, dtype):
    """Which operands are copied, not what is added up, goes by them."""
    def gradients(unpack):
        v = inputs(kind, dtype)
        with saved_tensors_hooks(lambda t: t.cpu(), lambda t: unpack(t.cuda())):
            y = call(kind, v)
        return torch.autograd.grad(y, list(v.values()), torch.ones_like(y))

    want = gradients(lambda t: t)
    for lay in (lambda t: torch.stack([t, t], -1)[..., 0], lambda t: t.t().contiguous().t() if t.dim() == 2 else t, part,
                lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)):
        assert all(torch.equal(a, e) for a, e in zip(gradients(lay), want))
