"""linear and gated_linear under tools that record the torch operations of a function to run them again: the launches of a native call are none
of them, so what was recorded would return memory that nothing has written."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import lmms_engine_amd as E

FUNCTIONS = {"linear": lambda x, w: E.linear(x, w, activation="silu"), "gated": lambda x, w: E.gated_linear(x, w, w)}


def traced(f, *args):
    return torch.jit.trace(f, args, check_trace=False)


def made(f, *args):
    return make_fx(f)(*args)


def made_before_dispatch(f, *args):
    return make_fx(f, pre_dispatch=True)(*args)


def without_values(f, *args):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(allow_non_fake_inputs=True):
        return f(*args)


RECORDERS = [traced, made, made_before_dispatch, without_values]


@pytest.mark.parametrize("record", RECORDERS)
@pytest.mark.parametrize("name", list(FUNCTIONS))
def test_recording_is_refused(name, record):
    """The refusal comes before any look at the tensors, so it needs no GPU."""
    with pytest.raises(NotImplementedError, match="recorded"):
        record(FUNCTIONS[name], torch.zeros(3, 8), torch.zeros(4, 8))


@pytest.mark.gpu
@pytest.mark.parametrize("record", RECORDERS)
@pytest.mark.parametrize("name", list(FUNCTIONS))
def test_recording_is_refused_on_a_gpu(name, record):
    x, w = torch.ones(3, 8, device="cuda"), torch.ones(4, 8, device="cuda")
    with pytest.raises(NotImplementedError, match="recorded"):
        record(FUNCTIONS[name], x, w)
    with pytest.raises(NotImplementedError, match="recorded"):
        record(lambda a, b: torch.autograd.grad(FUNCTIONS[name](a.requires_grad_(True), b).sum(), a)[0], x.clone(), w)
    assert torch.equal(FUNCTIONS[name](x, w), FUNCTIONS[name](x.clone(), w))  # and afterwards calls are taken again


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(FUNCTIONS))
def test_a_backward_pass_that_is_recorded_is_refused(name):
    x, w = torch.ones(3, 8, device="cuda", requires_grad=True), torch.ones(4, 8, device="cuda")
    y = FUNCTIONS[name](x, w)
    with pytest.raises(NotImplementedError, match="recorded"):
        make_fx(lambda dy: torch.autograd.grad(y, x, dy, retain_graph=True)[0])(torch.ones_like(y))
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.isfinite(dx).all()


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(FUNCTIONS))
def test_modes_that_watch_see_the_same_results(name):
    """Counters of operations and selective recomputation run what they see; calls inside give what they give outside."""
    from torch.utils.checkpoint import checkpoint, create_selective_checkpoint_contexts, CheckpointPolicy
    from torch.utils.flop_counter import FlopCounterMode

    g = torch.Generator(device="cuda").manual_seed(3)
    x, w = (torch.randn(*s, generator=g, device="cuda").requires_grad_(True) for s in ((6, 16), (8, 16)))

    def both(f):
        y = f(x, w)
        return [y.detach(), *torch.autograd.grad(y, (x, w), torch.ones_like(y))]

    want = both(FUNCTIONS[name])
    with FlopCounterMode(display=False):
        counted = both(FUNCTIONS[name])
    recomputed = both(lambda a, b: checkpoint(FUNCTIONS[name], a, b, use_reentrant=False))
    policy = lambda ctx, op, *args, **kwargs: CheckpointPolicy.PREFER_RECOMPUTE
    chosen = both(lambda a, b: checkpoint(FUNCTIONS[name], a, b, use_reentrant=False, context_fn=lambda: create_selective_checkpoint_contexts(policy)))
    for got in (counted, recomputed, chosen):
        assert all(torch.equal(a, e) for a, e in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
@pytest.mark.parametrize("name", list(FUNCTIONS))
def test_compiled_functions_break_their_graph_at_a_call(name, backend):
    g = torch.Generator(device="cuda").manual_seed(9)
    x, w = (torch.randn(*s, generator=g, device="cuda").requires_grad_(True) for s in ((6, 16), (8, 16)))

    def f(a, b):
        return FUNCTIONS[name](a * 2, b).relu() + 1

    def both(f):
        y = f(x, w)
        return [y.detach(), *torch.autograd.grad(y, (x, w), torch.ones_like(y))]

    for got, want in zip(both(torch.compile(f, backend=backend)), both(f)):
        assert torch.equal(got, want)
