"""What linear, gated_linear and the entry points behind them refuse, before anything is launched: no GPU needed."""
import ctypes
import itertools

import pytest
import torch

import lmms_engine_amd as E
from lmms_engine_amd import _abi, layers
from tests import layer_cases as cases


def test_cpu_tensors_and_wrong_arguments_are_refused():
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    with pytest.raises(_abi.MuonHipError, match="no CPU path"):
        E.linear(x, w)
    with pytest.raises(_abi.MuonHipError, match="no CPU path"):
        E.gated_linear(x, w, w)
    with pytest.raises(ValueError, match="activation is one of none, relu"):
        E.linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="activation is one of"):
        E.gated_linear(x, w, w, activation=None)
    with pytest.raises(TypeError):
        E.linear(x, w, None, "silu")  # the activation is named


class OnGpu(torch.Tensor):
    """A CPU tensor that says it is on a GPU: what is checked behind that, without one."""

    @property
    def is_cuda(self):
        return True


def gpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu)


@pytest.mark.parametrize("make,error,match", [
    (lambda: E.linear(gpu(2, 8), gpu(4, 9)), ValueError, "do not fit"),
    (lambda: E.linear(gpu(2, 8), gpu(8)), ValueError, "do not fit"),
    (lambda: E.linear(gpu(2, 8), gpu(4, 8).sum()), ValueError, "do not fit"),
    (lambda: E.linear(gpu(2, 8), gpu(4, 8).view(1, 4, 8)), ValueError, "do not fit"),
    (lambda: E.linear(gpu(2, 8).sum(), gpu(4, 8)), ValueError, "dimension"),
    (lambda: E.linear(gpu(2, 8), gpu(4, 8), gpu(1)), ValueError, "bias has shape"),
    (lambda: E.linear(gpu(2, 8), gpu(4, 8), gpu(1, 4)), ValueError, "bias has shape"),
    (lambda: E.linear(gpu(2, 8), gpu(4, 8), residual=gpu(4)), ValueError, "residual has shape"),
    (lambda: E.linear(gpu(2, 8), gpu(4, 8), residual=gpu(1, 4)), ValueError, "residual has shape"),
    (lambda: E.linear(gpu(2, 8), gpu(4, 8, dtype=torch.float32)), TypeError, "share one type"),
    (lambda: E.linear(gpu(2, 8), gpu(4, 8), gpu(4, dtype=torch.float32)), TypeError, "share one type"),
    (lambda: E.linear(gpu(2, 8, dtype=torch.float16), gpu(4, 8, dtype=torch.float16)), TypeError, "float32 and bfloat16"),
    (lambda: E.linear(gpu(2, 8, dtype=torch.int32), gpu(4, 8, dtype=torch.int32)), TypeError, "float32 and bfloat16"),
    (lambda: E.gated_linear(gpu(2, 8), gpu(4, 8), gpu(5, 8)), ValueError, "do not fit"),
    (lambda: E.gated_linear(gpu(2, 8), gpu(4, 8), gpu(4, 8), None, gpu(5)), ValueError, "bias has shape"),
    (lambda: E.gated_linear(gpu(2, 8), gpu(4, 8), torch.zeros(4, 8, dtype=torch.bfloat16)), _abi.MuonHipError, "no CPU path"),
])
def test_shapes_and_types_are_refused(make, error, match):
    with pytest.raises(error, match=match):
        make()


def valid(kind=0):
    p = _abi.Product(kind=kind, dtype=_abi.BF16, m=16, n=16, k=16)
    one = 1 << 20  # never read: every call below is refused
    for f in ("a", "b"):
        getattr(p, f)[:] = (one, one)
        getattr(p, f + "_row")[:] = (16, 16)
        getattr(p, f + "_col")[:] = (1, 1)
    p.out[:] = (one, one)
    return p


@pytest.mark.parametrize("kind,change,match", [
    (9, {}, "kind"),
    (-1, {}, "kind"),
    (0, dict(dtype=7), "dtype"),
    (0, dict(activation=6), "activation"),
    (0, dict(activation=-1), "activation"),
    (0, dict(m=-1), "negative"),
    (0, dict(k=-3), "negative"),
    (0, dict(a_row=(-16, 16)), "negative"),
    (2, dict(b_col=(1, -1)), "negative"),
    (0, dict(a=(None, None)), "null operand"),
    (1, dict(b=(1 << 20, None)), "null operand"),
    (2, dict(a=(1 << 20, None)), "null operand"),
    (3, dict(out=(1 << 20, None)), "null result"),
    (0, dict(aux=(None, 1 << 20)), "second results"),
    (1, dict(aux=(1 << 20, None)), "second results"),
    (1, dict(residual=1 << 20), "residual"),
    (0, dict(bias=(None, 1 << 20)), "two biases"),
    (2, dict(bias=(1 << 20, None)), "sums of products"),
    (3, dict(activation=3), "sums of products"),
    (2, dict(residual=1 << 20), "sums of products"),
])
def test_products_are_checked_before_any_launch(kind, change, match):
    lib, p = _abi.lib(), valid(kind)
    for name, v in change.items():
        if isinstance(v, tuple):
            getattr(p, name)[:] = v
        else:
            setattr(p, name, v)
    at = ctypes.addressof(p)
    assert lib.muon_hip_product_run(at, None, 0, None) == -1
    assert match in lib.muon_hip_last_error().decode()
    assert lib.muon_hip_product_workspace(at) == -1


def test_null_products_and_empty_results():
    lib = _abi.lib()
    assert lib.muon_hip_product_run(None, None, 0, None) == -1
    p = _abi.Product(kind=0, dtype=_abi.F32, m=0, n=5, k=3)
    assert lib.muon_hip_product_run(ctypes.addressof(p), None, 0, None) == 0  # nothing to write, nothing to read


def test_activation_gradients_are_checked_before_any_launch():
    lib, one = _abi.lib(), 1 << 20
    run = lib.muon_hip_act_grad
    assert run(one, 1, one, None, one, None, 8, None, None, 5, 4, 8, None, None) == -1  # dtype
    assert run(one, 1, one, None, one, None, 7, None, None, 1, 4, 8, None, None) == -1  # rows that overlap
    assert run(one, 1, one, None, one, one, 8, None, None, 1, 4, 8, None, None) == -1  # a second result of one factor
    assert run(one, 2, None, one, one, one, 8, None, None, 1, 4, 8, None, None) == -1  # a second factor alone
    assert run(one, 2, one, one, one, None, 8, None, None, 1, 4, 8, None, None) == -1  # one product of two
    assert run(one, 3, one, one, one, one, 8, None, None, 1, 4, 8, None, None) == -1
    assert run(None, 1, one, None, one, None, 8, None, None, 1, 4, 8, None, None) == -1
    assert run(one, 1, one, None, one, None, 8, one, None, 1, 4, 8, None, None) == -1  # sums without room for their parts
    assert lib.muon_hip_act_grad_partials(0, 5) == 0
    for m, n in ((1, 1), (65, 3), (5000, 4096), (100000, 20000)):
        floats = lib.muon_hip_act_grad_partials(m, n)
        assert floats > 0 and floats % n == 0 and floats * 4 <= 4 * n + m * n  # a part is a row of sums, at most one for eight rows
    assert lib.muon_hip_product_aux_bytes(_abi.BF16, 5, 7) == 105 and lib.muon_hip_product_aux_bytes(_abi.F32, 5, 7) == 140
    assert lib.muon_hip_product_aux_bytes(_abi.BF16, 1 << 30, 1 << 20) == 3 << 50
    assert lib.muon_hip_product_aux_bytes(9, 5, 7) < 0


def test_activation_names_are_those_of_the_header():
    assert layers.ACTIVATIONS == ("none", "relu", "sigmoid", "silu", "gelu", "gelu_tanh")


def product_of(kind, m, n, k, dtype=_abi.BF16, turned=(False, False), at=1 << 20):
    """A product of contiguous matrices, turned where the reduction runs down their columns; nothing is there to be read."""
    p = _abi.Product(kind=kind, dtype=dtype, m=m, n=n, k=k)
    for f, lines, turn in (("a", m, turned[0]), ("b", n, turned[1])):
        getattr(p, f)[:] = (at, at)
        getattr(p, f + "_row")[:] = (1, 1) if turn else (k, k)
        getattr(p, f + "_col")[:] = (lines, lines) if turn else (1, 1)
    p.out[:] = (1 << 20, 1 << 20)
    return p


MOST_THREADS = 2 ** 32 - 1  # of a launch


def test_no_launch_has_more_threads_than_a_grid_may_have():
    """Sizes up to the largest: a product is planned within the limit, or refused before anything is launched."""
    planned = 0
    big = [1, 7, 16, 250, 4096, 2 ** 20 + 1, 2 ** 24, 2 ** 27 - 16, 2 ** 27, 2 ** 28 + 5, 2 ** 30, 2 ** 31 - 70, 2 ** 31 - 1]
    for kind, dtype, m, n, k, turned, at in itertools.product(range(4), (_abi.BF16, _abi.F32), big, big, (1, 8, 33, 4096), itertools.product((False, True), repeat=2),
                                                              (1 << 20, (1 << 20) + 4)):
        try:
            r = _abi.product_route(product_of(kind, m, n, k, dtype, turned, at))
        except _abi.MuonHipError as e:
            assert "exceed one launch" in str(e)
            continue
        planned += 1
        assert 0 < r.groups * r.threads <= MOST_THREADS, (kind, dtype, m, n, k, turned, r.tile, r.parts, r.groups)
        assert r.copies <= MOST_THREADS and (r.copies > 0) == (max(r.a, r.b) >= _abi.OPERAND_ROWS_COPIED), (kind, dtype, m, n, k, turned, r.a, r.b, r.copies)
    assert planned > 1000


@pytest.mark.parametrize("kind", (_abi.PRODUCT_LINEAR, _abi.PRODUCT_GATED))
def test_a_few_rows_against_a_very_large_table(kind):
    """Where the walk over the weight has more workgroups than a launch, tiles take the call."""
    assert _abi.product_route(product_of(kind, 4, 2 ** 27 - 16, 64)).tile == 0
    for n in (2 ** 27, 2 ** 28, 2 ** 30 - 64):
        r = _abi.product_route(product_of(kind, 4, n, 64))
        assert r.tile > 0 and r.groups * r.threads <= MOST_THREADS, n


def test_activation_gradients_fit_a_launch():
    lib, one = _abi.lib(), 1 << 20
    for m, n in itertools.product((1, 9, 4096, 2 ** 24, 2 ** 30, 2 ** 31 - 1), (1, 255, 257, 4096, 2 ** 24, 2 ** 31 - 1)):
        chunks, rest = divmod(lib.muon_hip_act_grad_partials(m, n), n)
        assert rest == 0 and 1 <= chunks <= -(-m // 8)
        if chunks * -(-n // 256) * 256 > MOST_THREADS:
            assert m * n > 2 ** 50  # (a petabyte)
            assert lib.muon_hip_act_grad(one, 1, one, None, one, None, n, None, None, 1, m, n, None, None) == -2


def test_the_cases_run_every_kernel():
    """EVERY_KERNEL, which a GPU test runs, takes every tile of every type in every pass, over rows and over columns, whole and split, as 256
    compute units choose them: a rule that changes has to bring new cases."""
    ran = set()
    for dtype, t, k, n in cases.EVERY_KERNEL:
        for layer, xt, wt in itertools.product(cases.LAYERS, (False, True), (False, True)):
            for which, p in cases.products(layer, dtype, t, k, n, xt, wt).items():
                kernel, split = cases.kernel(p)
                parts, bk = _abi.product_route(p).parts, 64 if dtype == _abi.BF16 else 32
                if -(-p.k // bk) // parts >= 4:
                    ran.add((layer, which) + kernel + (split,))
    tiles = [(_abi.BF16, 64, 256), (_abi.BF16, 128, 256), (_abi.BF16, 128, 512), (_abi.BF16, 256, 512), (_abi.F32, 64, 256), (_abi.F32, 128, 256)]
    orders = {("linear", "forward"): [(0, 0), (0, 1), (1, 0), (1, 1)], ("gated", "forward"): [(0, 0), (1, 0)]}  # of the left and the right operand
    for (layer, which), split, tile in itertools.product(itertools.product(cases.LAYERS, ("forward", "dx", "dw")), (False, True), tiles):
        if layer == "linear" and split and tile == (_abi.BF16, 128, 256):
            continue  # (more tiles than compute units: one result of so many is not split)
        for a, b in orders.get((layer, which), [(int(which == "dw"), b) for b in (0, 1)]):
            assert (layer, which, *tile, a, b, layer == "gated" and which == "forward", split) in ran, (layer, which, tile, a, b, split)
