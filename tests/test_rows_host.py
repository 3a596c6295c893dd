"""What embedding, layer_norm, rms_norm, dropout and the entry points behind them refuse, before anything is launched, and the generator's published
numbers: no GPU needed."""
import ctypes

import pytest
import torch

import lmms_engine_amd as E
from lmms_engine_amd import _abi
from tests import rows_reference as R
from tests.test_layers_host import gpu
from tests.test_layers_recording import RECORDERS

ONE = 1 << 20  # an address that is never read: every call below is refused

CALLS = {"embedding": lambda x, w: E.embedding(torch.zeros(3, dtype=torch.int64), w), "layer_norm": lambda x, w: E.layer_norm(x, w[0]),
         "rms_norm": lambda x, w: E.rms_norm(x, residual=x), "dropout": lambda x, w: E.dropout(x, 0.1, seed=1)}


def test_the_generator_gives_its_published_numbers():
    """Known answers of Philox4x32-10, published with its paper."""
    full = 0xFFFFFFFF
    for c, key, want in (([0] * 4, 0, "6627e8d5e169c58dbc57ac4c9b00dbd8"), ([full] * 4, full << 32 | full, "408f276d41c83b0ea20bc7c66d5451fd"),
                         ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], 0x299F31D0 << 32 | 0xA4093822, "d16cfe0994fdcceb5001e42024126ea1")):
        assert "".join("%08x" % int(v) for v in R.philox(c, key)) == want


@pytest.mark.parametrize("name", list(CALLS))
def test_cpu_tensors_are_refused(name):
    with pytest.raises(_abi.MuonHipError, match="no CPU path"):
        CALLS[name](torch.zeros(2, 8), torch.zeros(4, 8))


@pytest.mark.parametrize("record", RECORDERS)
@pytest.mark.parametrize("name", list(CALLS))
def test_recording_is_refused(name, record):
    with pytest.raises(NotImplementedError, match="recorded"):
        record(CALLS[name], torch.zeros(3, 8), torch.zeros(4, 8))


def ids(*values, dtype=torch.int64):
    return torch.tensor(values, dtype=dtype).as_subclass(type(gpu(1)))


@pytest.mark.parametrize("make,error,match", [
    (lambda: E.embedding(ids(1), gpu(4)), ValueError, "weight has shape"),
    (lambda: E.embedding(ids(1), gpu(4, 8, 2)), ValueError, "weight has shape"),
    (lambda: E.embedding(ids(1, dtype=torch.int16), gpu(4, 8)), TypeError, "int32 or torch.int64"),
    (lambda: E.embedding(gpu(4), gpu(4, 8)), TypeError, "ids: "),
    (lambda: E.embedding(torch.tensor([1]), gpu(4, 8)), _abi.MuonHipError, "ids must live on a GPU"),
    (lambda: E.embedding(ids(1), gpu(4, 8, dtype=torch.float16)), TypeError, "float32 and bfloat16"),
    (lambda: E.embedding(ids(1), gpu(4, 8), padding_idx=4), ValueError, "padding_idx"),
    (lambda: E.embedding(ids(1), gpu(4, 8), padding_idx=-5), ValueError, "padding_idx"),
    (lambda: E.layer_norm(gpu(2, 8), gpu(7)), ValueError, "weight has shape"),
    (lambda: E.layer_norm(gpu(2, 8), gpu(8), gpu(1, 8)), ValueError, "bias has shape"),
    (lambda: E.layer_norm(gpu(2, 8), gpu(8, dtype=torch.float32)), TypeError, "share one type"),
    (lambda: E.layer_norm(gpu(2, 8), residual=gpu(8)), ValueError, "residual has shape"),
    (lambda: E.layer_norm(gpu(2, 8), eps=-1.0), ValueError, "eps"),
    (lambda: E.layer_norm(gpu(2, 8), eps=float("nan")), ValueError, "eps"),
    (lambda: E.layer_norm(gpu(2, 8).sum()), ValueError, "dimension"),
    (lambda: E.rms_norm(gpu(2, 8, dtype=torch.float16)), TypeError, "float32 and bfloat16"),
    (lambda: E.rms_norm(gpu(2, 8), torch.zeros(8, dtype=torch.bfloat16)), _abi.MuonHipError, "no CPU path"),
    (lambda: E.dropout(gpu(2, 8), 1.5, seed=1), ValueError, "p is 1.5"),
    (lambda: E.dropout(gpu(2, 8), float("nan"), seed=1), ValueError, "p is nan"),
    (lambda: E.dropout(gpu(2, 8), 0.1, seed=2 ** 64), ValueError, "64 bits"),
    (lambda: E.dropout(gpu(2, 8), 0.1, seed=-2 ** 63 - 1), ValueError, "64 bits"),
    (lambda: E.dropout(gpu(2, 8), 0.1, seed=1, site=2 ** 32), ValueError, "32 bits"),
    (lambda: E.dropout(gpu(2, 8), 0.1, seed=1, site=-1), ValueError, "32 bits"),
    (lambda: E.dropout(gpu(2, 8), 0.1, seed=ids(1, 2)), ValueError, "seed has shape"),
    (lambda: E.dropout(gpu(2, 8), 0.1, seed=ids(1, dtype=torch.int32)), TypeError, "seed: "),
    (lambda: E.dropout(gpu(2, 8), 0.1, seed=torch.tensor([1])), _abi.MuonHipError, "seed must live on a GPU"),
    (lambda: E.dropout(gpu(2, 8), 0.1), TypeError, "seed"),
    (lambda: E.dropout(gpu(2, 8), 0.1, seed=1.5), TypeError, "integer"),
    (lambda: E.dropout(gpu(2, 8), 0.1, seed="1"), TypeError, "integer"),
    (lambda: E.dropout(gpu(2, 8), 0.1, seed=1, residual=gpu(2, 1)), ValueError, "residual has shape"),
    (lambda: E.dropout(gpu(2, 8), 0.1, seed=1), NotImplementedError, "OnGpu"),
])
def test_shapes_and_types_are_refused(make, error, match):
    with pytest.raises(error, match=match):
        make()


def norm(**change):
    p = _abi.Norm(kind=_abi.NORM_LAYER, dtype=_abi.BF16, rows=4, n=8, x=ONE, x_row=8, weight=ONE, bias=ONE, eps=1e-5, y=ONE)
    for name, v in change.items():
        setattr(p, name, v)
    return p


@pytest.mark.parametrize("change,code,match", [
    (dict(kind=2), -1, "kind"), (dict(dtype=9), -1, "dtype"), (dict(rows=-1), -1, "size"), (dict(n=-1), -1, "size"), (dict(n=0x7fffffff), -2, "the most"),
    (dict(kind=_abi.NORM_RMS), -1, "no bias"), (dict(eps=-1e-9), -1, "eps"), (dict(eps=float("nan")), -1, "eps"), (dict(x=None), -1, "null"),
    (dict(y=None), -1, "null"), (dict(residual=ONE, res_row=8), -1, "together"), (dict(sum=ONE), -1, "together"), (dict(x_row=7), -1, "overlap"),
    (dict(residual=ONE, res_row=0, sum=ONE), -1, "overlap"),
])
def test_norms_are_checked_before_any_launch(change, code, match):
    lib, p = _abi.lib(), norm(**change)
    assert lib.muon_hip_norm_run(ctypes.addressof(p), None) == code
    assert match in lib.muon_hip_last_error().decode()


def kernel(kind, dtype, rows, n, backward):
    r = _abi.norm_route(kind, dtype, rows, n, backward)
    # lanes below a wave's are a kernel of their own, which has one piece
    single = n < (4 if dtype == _abi.F32 else 8)  # rows of less than a piece
    return (kind, dtype, backward, r.pieces) + ((bool(r.ragged), r.lanes < 64, single) if r.pieces else ())


def test_the_gpu_tests_run_every_kernel_of_the_norms():
    from tests.test_gpu_rows import COLUMNS, MANY_ROWS, ROWS_OF

    cases = [(m, n) for n in COLUMNS for m in ROWS_OF(n)] + MANY_ROWS
    sizes = [(m, n) for m in (1, 70, 2000, 5000, 300000) for n in list(range(1, 200)) + list(range(200, 40000, 37)) + [2 ** i for i in range(17)]]
    for kind in (_abi.NORM_LAYER, _abi.NORM_RMS):
        for dtype in (_abi.F32, _abi.BF16):
            for backward in (False, True):
                ran, there_are = ({kernel(kind, dtype, m, n, backward) for m, n in some} for some in (cases, sizes))
                assert there_are <= ran, there_are - ran
                assert len(there_are) >= 7


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("dtype", [_abi.F32, _abi.BF16])
def test_norms_are_laid_over_whole_rows_and_launches(dtype, backward):
    piece = 4 if dtype == _abi.F32 else 8
    for kind in (_abi.NORM_LAYER, _abi.NORM_RMS):
        for n in list(range(1, 300)) + [1000, 4096, 8200, 16384, 16385, 32769, 70001, 0x7fffffff - (1 << 20)]:
            for rows in (1, 9, 4097, 0x7fffffff):
                r = _abi.norm_route(kind, dtype, rows, n, backward)
                assert 0 < r.groups * r.threads < 2 ** 32 and r.threads % 64 == 0 and r.threads <= 1024
                if r.pieces:
                    assert r.lanes * r.pieces * (piece if n >= piece else 1) >= n and r.lanes <= r.threads and bool(r.ragged) == (n > piece and n % piece != 0)
                    assert r.lanes % 64 == 0 or (r.lanes in (8, 16, 32) and r.pieces == 1)
                    if backward:  # the columns' sums of several rows at once meet in LDS
                        assert r.threads <= max(r.lanes, 64) or 4 * n <= 64 * 1024
                if backward:
                    assert r.groups <= 1024
    lib = _abi.lib()
    out = _abi.NormRoute()
    assert lib.muon_hip_route_norm(3, dtype, 4, 8, 0, 256, ctypes.addressof(out)) == -1
    assert lib.muon_hip_route_norm(0, 5, 4, 8, 0, 256, ctypes.addressof(out)) == -1
    assert lib.muon_hip_route_norm(0, dtype, 4, 8, 0, 0, ctypes.addressof(out)) == -1
    assert lib.muon_hip_route_norm(0, dtype, 4, 8, 0, 256, None) == -1


def norm_grad(**change):
    p = _abi.NormGrad(kind=_abi.NORM_LAYER, dtype=_abi.BF16, rows=4, n=8, dy=ONE, dy_row=8, s=ONE, s_row=8, weight=ONE, stats=ONE, dx=ONE, dweight=ONE, dbias=ONE)
    for name, v in change.items():
        setattr(p, name, v)
    return p


@pytest.mark.parametrize("change,code,match", [
    (dict(kind=-1), -1, "kind"), (dict(dtype=2), -1, "dtype"), (dict(rows=-1), -1, "size"), (dict(n=0x7fffffff), -2, "the most"), (dict(dy=None), -1, "null"),
    (dict(s=None), -1, "null"), (dict(stats=None, dx=None), -1, "null"), (dict(dy_row=7), -1, "overlap"), (dict(s_row=-8), -1, "overlap"),
    (dict(ds=ONE, ds_row=1), -1, "overlap"), (dict(kind=_abi.NORM_RMS), -1, "no bias"),
])
def test_gradients_of_norms_are_checked_before_any_launch(change, code, match):
    lib, p = _abi.lib(), norm_grad(**change)
    assert lib.muon_hip_norm_grad_run(ctypes.addressof(p), ONE, 1 << 40, None) == code
    assert match in lib.muon_hip_last_error().decode()
    assert lib.muon_hip_norm_grad_workspace(ctypes.addressof(p)) == code


def test_embeddings_are_checked_before_any_launch():
    lib = _abi.lib()

    def look_up(ids=ONE, tokens=3, table=ONE, row=8, vocab=5, n=8, dtype=1, out=ONE):
        return lib.muon_hip_embedding(ids, 1, tokens, table, row, vocab, n, dtype, 1.0, out, None)

    for bad in (dict(ids=None), dict(table=None), dict(row=7), dict(tokens=-1), dict(vocab=-1), dict(n=-1), dict(dtype=3), dict(out=None), dict(vocab=0x7fffffff)):
        assert look_up(**bad) == -1, bad
    assert look_up(n=0x7fffffff) == -2
    assert look_up(tokens=0, ids=None, out=None) == 0 and look_up(n=0, out=None) == 0

    def grad(ids=ONE, tokens=3, dy=ONE, row=8, vocab=5, n=8, dtype=1, skip=-1, out=ONE, room=1 << 40):
        return lib.muon_hip_embedding_grad(ids, 1, tokens, dy, row, vocab, n, dtype, 1.0, skip, out, ONE, room, None)

    for bad in (dict(ids=None), dict(dy=None), dict(row=7), dict(tokens=-1), dict(vocab=-1), dict(n=-1), dict(dtype=3), dict(out=None), dict(skip=5), dict(skip=-2)):
        assert grad(**bad) == -1, bad
    assert grad(vocab=0, out=None) == 0 and grad(n=0, out=None) == 0
    assert lib.muon_hip_embedding_grad_workspace(-1, 5, 8, 1) == -1 and lib.muon_hip_embedding_grad_workspace(3, -5, 8, 1) == -1


def test_dropouts_are_checked_before_any_launch():
    lib = _abi.lib()

    def drop(x=ONE, y=ONE, count=8, dtype=1, p=0.5):
        return lib.muon_hip_dropout(x, None, y, count, dtype, p, 1, None, 0, None)

    for bad in (dict(x=None), dict(y=None), dict(count=-1), dict(dtype=2), dict(p=-0.1), dict(p=1.1), dict(p=float("nan"))):
        assert drop(**bad) == -1, bad
    assert drop(count=0, x=None, y=None) == 0
