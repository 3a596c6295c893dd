"""What embedding, layer_norm, rms_norm and dropout keep for their backward pass, when it is not there any more, or not what it was."""
import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks

import lmms_engine_amd as E

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16]


def part(values):
    """The values behind others of their memory: what is left of their address once that is freed is not null."""
    return torch.cat([values.flatten()[:1].expand(16), values.flatten()])[16:].view(values.shape)


def leaf(*shape, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(len(shape))
    return part(1 + torch.randn(shape, generator=g, device=DEV).to(dtype)).requires_grad_(True)


def free(t):
    t.untyped_storage().resize_(0)


# Calls on x [6, 40], r like it and w [40]: (result, what it is differentiated by, what is freed).
def weight(x, r, w):
    return E.layer_norm(x, w), x, w


def weight_beside_a_residual(x, r, w):
    return E.rms_norm(x, w, residual=r)[0], r, w


def summed(x, r, w):
    y, s = E.layer_norm(x, w, residual=r)
    return y, x, s


def summed_for_the_weight(x, r, w):
    y, s = E.rms_norm(x, w, residual=r)
    return y, w, s


def input_for_the_weight(x, r, w):
    a = x.detach().clone()
    return E.layer_norm(a, w), w, a


def ids(x, r, w):
    i = part(torch.tensor([0, 3, 3], device=DEV))
    return E.embedding(i, x), x, i


def seed(x, r, w):
    s = part(torch.tensor([7], device=DEV))
    return E.dropout(x, 0.5, seed=s), x, s


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("call", [weight, weight_beside_a_residual, summed, summed_for_the_weight, input_for_the_weight, ids, seed])
def test_memory_that_was_freed_is_not_taken_for_what_was_left_out(call, dtype):
    """Nor is it read: a version counter does not tell that it is gone."""
    y, of, gone = call(leaf(6, 40, dtype=dtype), leaf(6, 40, dtype=dtype), leaf(40, dtype=dtype))
    free(gone)
    with pytest.raises(ValueError, match="freed"):
        torch.autograd.grad(y, of, torch.ones_like(y))


@pytest.mark.parametrize("call", [weight, summed, ids, seed])
def test_an_incoming_gradient_that_was_freed(call):
    y, of, _ = call(leaf(6, 40), leaf(6, 40), leaf(40))
    dy = part(torch.ones_like(y))
    free(dy)
    with pytest.raises(ValueError, match="freed"):
        torch.autograd.grad(y, of, dy)


def test_what_a_gradient_does_not_read_may_be_gone():
    """A norm's weight is read for the input's gradient alone, its input for all but the bias', a dropout's input by none."""
    x, r, w, b = leaf(6, 40), leaf(6, 40), leaf(40), leaf(40)
    dy, ds = torch.randn(6, 40, device=DEV), torch.randn(6, 40, device=DEV)
    want = torch.autograd.grad(E.layer_norm(x, w, b, residual=r), (w, b), (dy, ds))
    y, s = E.layer_norm(x, w, b, residual=r)
    free(w)
    assert all(torch.equal(a, e) for a, e in zip(torch.autograd.grad((y, s), (w, b), (dy, ds), retain_graph=True), want))
    free(s)
    (db,) = torch.autograd.grad(y, b, dy)
    # either sum adds six values, in an order of its own
    assert ((db - want[1]).abs() <= 2 * 6 * 2.0 ** -24 * dy.abs().sum(0)).all()
    y = E.dropout(x, 0.5, seed=3, residual=r)
    free(x)
    assert torch.equal(torch.autograd.grad(y, r, dy)[0], dy)


def kept_by(call, dtype):
    """The tensors that a call keeps, as hooks see them."""
    kept = []
    with saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        call(leaf(6, 40, dtype=dtype), leaf(6, 40, dtype=dtype), leaf(40, dtype=dtype))
    return len(kept)


CALLS = [weight, weight_beside_a_residual, input_for_the_weight, ids, seed]
OTHERS = {
    "a type": (lambda t: t.to(torch.float16 if t.is_floating_point() else torch.int16), TypeError),
    "a wider type": (lambda t: t.double(), TypeError),
    "a device": (lambda t: t.cpu(), ValueError),
    "fewer values": (lambda t: t.flatten()[:0], ValueError),
    "a shape": (lambda t: torch.stack([t, t]), ValueError),
    "a layout": (lambda t: t.to_sparse(), NotImplementedError),
}


@pytest.mark.parametrize("other", list(OTHERS))
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("call", CALLS)
def test_what_hooks_give_back_is_what_was_kept(call, dtype, other):
    change, error = OTHERS[other]
    count = kept_by(call, dtype)
    assert count == {"ids": 1, "seed": 1, "input_for_the_weight": 2}.get(call.__name__, 3)
    for i in range(count):
        seen = []
        with saved_tensors_hooks(lambda t: seen.append(t) or (len(seen) - 1, t), lambda p: change(p[1]) if p[0] == i else p[1]):
            y, of, _ = call(leaf(6, 40, dtype=dtype), leaf(6, 40, dtype=dtype), leaf(40, dtype=dtype))
        with pytest.raises(error, match="kept for a backward pass"):
            torch.autograd.grad(y, of, torch.ones_like(y))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("call", CALLS)
def test_hooks_may_give_back_other_strides_and_addresses(call, dtype):
    def gradient(unpack):
        with saved_tensors_hooks(lambda t: t.cpu(), lambda t: unpack(t.cuda())):
            y, of, _ = call(leaf(6, 40, dtype=dtype), leaf(6, 40, dtype=dtype), leaf(40, dtype=dtype))
        return torch.autograd.grad(y, of, torch.ones_like(y))[0]

    want = gradient(lambda t: t)
    for lay in (lambda t: torch.stack([t, t], -1)[..., 0], lambda t: t.t().contiguous().t() if t.dim() == 2 else t, part):
        assert torch.equal(gradient(lay), want)


@pytest.mark.parametrize("call", CALLS)
def test_incoming_gradients_that_are_no_plain_tensors_raise(call):
    y, of, _ = call(leaf(6, 40), leaf(6, 40), leaf(40))
    for dy, batched in ((torch.ones_like(y).to_sparse(), False), (torch.ones(3, *y.shape, device=DEV), True)):
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, of, dy, is_grads_batched=batched, retain_graph=True)
