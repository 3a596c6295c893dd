"""What linear and gated_linear keep for their backward pass, when it is not there any more."""
import pytest
import torch

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
