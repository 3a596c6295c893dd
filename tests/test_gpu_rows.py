"""embedding, layer_norm, rms_norm and dropout against their formulas in 64 bits (rows_reference.py)."""
import ctypes

import numpy as np
import pytest
import torch

from torch.fx.experimental.proxy_tensor import make_fx

import lmms_engine_amd as E
from lmms_engine_amd import _abi
from tests import rows_reference as R
from tests.test_layers_recording import RECORDERS

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
DTYPES = [F32, BF16]


def gen_of(*key):
    return torch.Generator(device=DEV).manual_seed(sum((i + 1) * ord(c) for i, c in enumerate(repr(key))))


def rnd(g, *shape, scale=1.0, dtype=F32):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


# ---- norms ------------------------------------------------------------------------------------------


def run_norm(kind, x, w, b, r, eps, dy, ds, wants="xwbr"):
    """{name: result} of a call and of its backward pass."""
    leaf = {"x": x, "w": w, "b": b, "r": r}
    named = {k: v.detach().requires_grad_(k in wants) for k, v in leaf.items() if v is not None}
    if kind == "layer":
        out = E.layer_norm(named["x"], named.get("w"), named.get("b"), eps=eps, residual=named.get("r"))
    else:
        out = E.rms_norm(named["x"], named.get("w"), eps=eps, residual=named.get("r"))
    y, s = out if r is not None else (out, None)
    asked = {k: v for k, v in named.items() if v.requires_grad}
    got = {"y": y.detach(), "s": None if s is None else s.detach()}
    if asked:
        outs, incoming = ([y, s], [dy, ds]) if s is not None and s.requires_grad else ([y], [dy])
        got.update({"d" + k: g for k, g in zip(asked, torch.autograd.grad(outs, list(asked.values()), incoming))})
    return got


def compare_norm(kind, x, w, b, r, eps, dy, ds, got):
    dtype, wide = x.dtype, lambda t: None if t is None else t.detach().double()
    s = wide(x)
    if r is not None:
        R.check("s", got["s"], s + wide(r), R.F * (s + wide(r)).abs(), dtype)
        s = wide(got["s"])  # what is normalised
    R.check("y", got["y"], *R.norm(kind, s, wide(w), wide(b), eps)["y"], dtype)
    with_ds = wide(ds) if r is not None and ("dx" in got or "dr" in got) else None
    want = R.norm_grad(kind, s, wide(w), eps, wide(dy), with_ds)
    for name in ("dx", "dr", "dw", "db"):
        if name in got:
            R.check(name, got[name], *want["dx" if name == "dr" else name], dtype)


# columns: one, less than a piece, whole pieces and odd ones, every number of lanes to a row, more than fits into registers; test_rows_host.py holds these
# lists to running every kernel
COLUMNS = [1, 5, 8, 12, 64, 100, 128, 251, 256, 500, 896, 1024, 1028, 2047, 2048, 4096, 4100, 6144, 8192, 12288, 10001, 2502, 5005, 16381, 16384, 20000, 24577, 33000, 70001]


def ROWS_OF(n):
    return (1, 3, 70 if n < 20000 else 5)


@pytest.mark.parametrize("n", COLUMNS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_norms_of_all_widths(kind, dtype, n):
    for rows in ROWS_OF(n):
        g = gen_of(kind, dtype, n, rows)
        print(kind, dtype, rows, n, flush=True)
        x, r, dy, ds = (rnd(g, rows, n, dtype=dtype) for _ in range(4))
        x = (x + 0.3).to(dtype)
        w, b = (1 + rnd(g, n, scale=0.3)).to(dtype), rnd(g, n, scale=0.1, dtype=dtype)
        for weight, bias, residual in ((w, b, r), (w, None, None), (None, b, r), (None, None, None)):
            bias = bias if kind == "layer" else None
            got = run_norm(kind, x, weight, bias, residual, 1e-5, dy, ds)
            compare_norm(kind, x, weight, bias, residual, 1e-5, dy, ds, got)


MANY_ROWS = [(777, 251), (2100, 128), (5000, 80), (1030, 1024), (1500, 4096), (600, 2056), (300, 8192), (4200, 2048), (2100, 4090), (4200, 1000)]


@pytest.mark.parametrize("rows,n", MANY_ROWS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_norms_of_many_rows(kind, dtype, rows, n):
    g = gen_of(kind, dtype, n, rows)
    x, r, dy, ds = (rnd(g, rows, n, dtype=dtype) for _ in range(4))
    w, b = (1 + rnd(g, n, scale=0.3)).to(dtype), rnd(g, n, scale=0.1, dtype=dtype) if kind == "layer" else None
    for residual in (r, None):
        got = run_norm(kind, x, w, b, residual, 1e-6, dy, ds)
        compare_norm(kind, x, w, b, residual, 1e-6, dy, ds, got)
        again = run_norm(kind, x, w, b, residual, 1e-6, dy, ds)
        assert all(torch.equal(got[k], again[k]) for k in got if got[k] is not None)  # sums have one order


@pytest.mark.parametrize("wants", ["x", "w", "b", "r", "wb", "xw", "xb", "br", "xr", "wr"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_each_gradient_by_itself(dtype, wants):
    g = gen_of(dtype, wants)
    rows, n = 67, 264
    x, r, dy, ds = (rnd(g, rows, n, dtype=dtype) for _ in range(4))
    w, b = (1 + rnd(g, n, scale=0.3)).to(dtype), rnd(g, n, scale=0.1, dtype=dtype)
    for kind in ("layer", "rms"):
        mine = wants if kind == "layer" else wants.replace("b", "")
        if mine:
            got = run_norm(kind, x, w, b if kind == "layer" else None, r, 1e-5, dy, ds, mine)
            assert set(got) == {"y", "s"} | {"d" + k for k in mine}
            compare_norm(kind, x, w, b if kind == "layer" else None, r, 1e-5, dy, ds, got)


LAYOUTS = {
    "columns first": lambda g, m, n, d: rnd(g, n, m, dtype=d).t(),
    "rows apart": lambda g, m, n, d: rnd(g, m, n + 13, dtype=d)[:, 5:5 + n],
    "every other row": lambda g, m, n, d: rnd(g, 2 * m, n, dtype=d)[::2],
    "rows backwards": lambda g, m, n, d: rnd(g, m, n, dtype=d).flip(0),
    "one row for all": lambda g, m, n, d: rnd(g, 1, n, dtype=d).expand(m, n),
    "one value for a row": lambda g, m, n, d: rnd(g, m, 1, dtype=d).expand(m, n),
    "three dimensions": lambda g, m, n, d: rnd(g, 5, m // 5, n, dtype=d),
    "heads of tokens": lambda g, m, n, d: rnd(g, m // 5, 7 * n, dtype=d)[:, n:6 * n].view(m // 5, 5, n),
    "heads first": lambda g, m, n, d: rnd(g, m // 5, 5, n, dtype=d).transpose(0, 1),
}


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("dtype", DTYPES)
def test_norms_of_any_layout(dtype, layout):
    make = LAYOUTS[layout]
    for m, n in ((40, 64), (35, 77)):
        g = gen_of(dtype, layout, m, n)
        x, r, dy, ds = (make(g, m, n, dtype) for _ in range(4))
        w, b = rnd(g, 2 * n, dtype=dtype)[::2], rnd(g, n + 1, dtype=dtype)[1:]
        if layout == "one value for a row":
            dy, ds = (rnd(g, m, n, dtype=dtype) for _ in range(2))
            x = x + rnd(g, m, n, dtype=dtype)
        for kind in ("layer", "rms"):
            bias = b if kind == "layer" else None
            for residual in (r, None):
                got = run_norm(kind, x, w, bias, residual, 1e-5, dy, ds)
                assert got["y"].is_contiguous() and got["y"].shape == x.shape
                compare_norm(kind, x, w, bias, residual, 1e-5, dy, ds, got)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_norms(dtype, kind):
    for shape in ((0, 16), (3, 0), (0, 0), (2, 0, 8)):
        x, r = (torch.zeros(*shape, dtype=dtype, device=DEV).requires_grad_(True) for _ in range(2))
        w, b = (torch.ones(shape[-1], dtype=dtype, device=DEV).requires_grad_(True) for _ in range(2))
        y, s = E.layer_norm(x, w, b, residual=r) if kind == "layer" else E.rms_norm(x, w, residual=r)
        assert y.shape == s.shape == x.shape
        named = (x, w, r) + ((b,) if kind == "layer" else ())
        for t, d in zip(named, torch.autograd.grad([y, s], named, [torch.ones_like(y), torch.ones_like(s)])):
            assert d.shape == t.shape and bool((d == 0).all())  # a sum over no rows


def test_the_sum_alone_or_the_norm_alone_is_differentiated():
    g = gen_of("alone")
    x, r, dy = (rnd(g, 9, 40, dtype=BF16) for _ in range(3))
    w, b = rnd(g, 40, dtype=BF16), rnd(g, 40, dtype=BF16)
    leaves = [t.requires_grad_(True) for t in (x, r, w, b)]
    y, s = E.layer_norm(x, w, b, residual=r)
    dx, dr, dw, db = torch.autograd.grad(s, leaves, dy)
    assert torch.equal(dx, dy) and torch.equal(dr, dy) and not dw.any() and not db.any()
    y, s = E.layer_norm(x, w, b, residual=r)
    got = torch.autograd.grad(y, leaves, dy)
    y, s = E.layer_norm(x, w, b, residual=r)
    want = torch.autograd.grad([y, s], leaves, [dy, torch.zeros_like(dy)])
    assert all(torch.equal(a, e) for a, e in zip(got, want))


def test_a_frozen_stream_is_not_differentiated():
    g = gen_of("frozen")
    x, r, w = rnd(g, 4, 32), rnd(g, 4, 32), rnd(g, 32).requires_grad_(True)
    y, s = E.rms_norm(x, w, residual=r)
    assert y.requires_grad and not s.requires_grad
    assert not E.rms_norm(x, w.detach(), residual=r)[0].requires_grad
    with torch.no_grad():
        assert not E.rms_norm(x, w, residual=r)[0].requires_grad


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_values_that_are_no_numbers_stay_in_their_rows(kind, dtype):
    g = gen_of(kind, dtype)
    for n in (64, 261, 4096):
        x, dy, ds = rnd(g, 12, n, dtype=dtype), rnd(g, 12, n, dtype=dtype), rnd(g, 12, n, dtype=dtype)
        w = (1 + rnd(g, n, scale=0.2)).to(dtype)
        want = run_norm(kind, x, w, None, torch.zeros_like(x), 1e-5, dy, ds, "x")
        bad = x.clone()
        bad[1, n - 1], bad[4, 3], bad[7, 5] = float("nan"), float("inf"), float("-inf")
        got = run_norm(kind, bad, w, None, torch.zeros_like(x), 1e-5, dy, ds, "x")
        rest = [i for i in range(12) if i not in (1, 4, 7)]
        for name in ("y", "s", "dx"):
            assert torch.equal(got[name][rest], want[name][rest])
        assert torch.isnan(got["y"][1]).all() and torch.isnan(got["dx"][1]).all()
        assert torch.isnan(got["y"][4, 3]) and torch.isnan(got["y"][7, 5])


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_one_value_and_rows_far_from_zero(dtype):
    g = gen_of("constant", dtype)
    x = torch.full((3, 300), 2.5, dtype=dtype, device=DEV)
    assert not E.layer_norm(x, eps=1e-5).any()
    assert not E.rms_norm(torch.zeros_like(x), eps=1e-6).any()
    far = (100.0 + rnd(g, 40, 1000, scale=2.0)).to(dtype)
    dy = rnd(g, 40, 1000, dtype=dtype)
    got = run_norm("layer", far, None, None, None, 1e-5, dy, None)
    compare_norm("layer", far, None, None, None, 1e-5, dy, None, got)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_gradients_against_differences(kind):
    """The derivative along a direction is what a small step along it changes, to the second order of the step (fp32: 1e-3 of it)."""
    g = gen_of(kind, "differences")
    x, r, dy, ds = (rnd(g, 6, 96).double() for _ in range(4))
    w, b = 1 + rnd(g, 96, scale=0.3).double(), rnd(g, 96).double()

    def loss(x, r, w, b):
        out = E.layer_norm(x.float(), w.float(), b.float(), residual=r.float()) if kind == "layer" else E.rms_norm(x.float(), w.float(), residual=r.float())
        return (out[0].double() * dy + out[1].double() * ds).sum()

    got = run_norm(kind, x.float(), w.float(), b.float() if kind == "layer" else None, r.float(), 1e-5 if kind == "layer" else 1e-6, dy.float(), ds.float())
    point = [x.float().double(), r.float().double(), w.float().double(), b.float().double()]
    for i, name in enumerate(("dx", "dr", "dw", "db")):
        if name not in got:
            continue
        step = rnd(g, *point[i].shape).double() * 2.0 ** -6
        ahead, back = ([p + sign * step if j == i else p for j, p in enumerate(point)] for sign in (1, -1))
        change = (loss(*ahead) - loss(*back)) / 2
        along = (got[name].double() * step).sum()
        size = (got[name].double().abs() * step.abs()).sum()
        # third derivatives of a norm of values around 1 times step^2 (2^-12), and the fp32 of either loss
        assert abs(change - along) <= 4e-3 * size, (name, change.item(), along.item(), size.item())


# ---- embedding --------------------------------------------------------------------------------------

IDS = {
    "any": lambda g, t, v: torch.randint(0, v, (t,), generator=g, device=DEV),
    "one": lambda g, t, v: torch.full((t,), v - 1, device=DEV),
    "runs": lambda g, t, v: torch.arange(t, device=DEV) // 37 % v,
    "most of one": lambda g, t, v: torch.where(torch.rand(t, generator=g, device=DEV) < 0.7, v // 2, torch.randint(0, v, (t,), generator=g, device=DEV)),
    "each once": lambda g, t, v: torch.randperm(max(t, v), generator=g, device=DEV)[:t] % v,
    "outside too": lambda g, t, v: torch.randint(-v, 2 * v, (t,), generator=g, device=DEV),
}


def run_embedding(ids, w, dy, scale=1.0, padding_idx=None):
    w = w.detach().requires_grad_(True)
    y = E.embedding(ids, w, scale=scale, padding_idx=padding_idx)
    return y.detach(), torch.autograd.grad(y, w, dy)[0]


def compare_embedding(ids, w, dy, scale, padding_idx, y, dw):
    vocab, n = w.shape
    known = (ids >= 0) & (ids < vocab)
    want = w.double()[ids.clamp(0, vocab - 1).long()] * scale
    want[~known] = float("nan")
    R.check("y", y, want, (0 if scale == 1 else 2 * R.F) * want.abs(), w.dtype if scale != 1 else None)
    skip = -1 if padding_idx is None else padding_idx % vocab
    dw_want, error = R.embedding_grad(ids.reshape(-1), dy.double().reshape(-1, n), vocab, scale, skip)
    R.check("dw", dw, dw_want, error, w.dtype)


@pytest.mark.parametrize("ids", list(IDS))
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,vocab,n", [(1, 1, 1), (1, 50, 4096), (7, 5, 12), (300, 17, 64), (513, 1000, 251), (2000, 3000, 1024), (4099, 77, 130),
                                            (9000, 20011, 96), (20001, 513, 264), (140000, 4000, 40)])
def test_embeddings(tokens, vocab, n, dtype, ids):
    g = gen_of(tokens, vocab, n, dtype, ids)
    print(tokens, vocab, n, dtype, ids, flush=True)
    at = IDS[ids](g, tokens, vocab)
    w, dy = rnd(g, vocab, n, dtype=dtype), rnd(g, tokens, n, dtype=dtype)
    scale = 1.0 if tokens % 2 else n ** 0.5
    padding = None if tokens % 3 else -1
    y, dw = run_embedding(at, w, dy, scale, padding)
    compare_embedding(at, w, dy, scale, padding, y, dw)
    y32, dw32 = run_embedding(at.int(), w, dy, scale, padding)
    assert torch.equal(y.nan_to_num(), y32.nan_to_num()) and torch.equal(dw, dw32)  # whichever type ids have, and the same bits again


@pytest.mark.parametrize("dtype", DTYPES)
def test_embeddings_of_any_layout(dtype):
    g = gen_of("layouts", dtype)
    ids = torch.randint(0, 30, (6, 14), generator=g, device=DEV)
    for n in (64, 51):
        for w in (rnd(g, n, 30, dtype=dtype).t(), rnd(g, 60, n + 3, dtype=dtype)[::2, 1:1 + n], rnd(g, 1, n, dtype=dtype).expand(30, n)):
            for i in (ids, ids.t(), ids[:, ::2], ids[0, 0], ids[2:2], ids.view(2, 3, 2, 7)):
                dy = rnd(g, n, *i.shape, dtype=dtype).movedim(0, -1)
                y, dw = run_embedding(i, w, dy)
                assert y.shape == (*i.shape, n) and dw.shape == w.shape
                compare_embedding(i, w, dy, 1.0, None, y, dw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_embeddings(dtype):
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    w = torch.ones(5, 8, dtype=dtype, device=DEV).requires_grad_(True)
    y = E.embedding(none, w)
    assert y.shape == (0, 8) and not torch.autograd.grad(y, w, torch.zeros_like(y))[0].any()
    y = E.embedding(torch.tensor([0, 3], device=DEV), torch.ones(0, 8, dtype=dtype, device=DEV))
    assert y.shape == (2, 8) and torch.isnan(y).all()
    assert E.embedding(torch.tensor([0, 3], device=DEV), torch.ones(4, 0, dtype=dtype, device=DEV)).shape == (2, 0)


def test_rows_without_tokens_hide_nothing():
    """Gradients that are no numbers reach the rows of their ids alone."""
    g = gen_of("nan")
    ids = torch.randint(0, 40, (500,), generator=g, device=DEV)
    dy = rnd(g, 500, 72, dtype=BF16)
    ids[13], ids[400] = 40, 41
    dy[13], dy[400, 5] = float("nan"), float("inf")
    w = rnd(g, 60, 72, dtype=BF16)
    _, dw = run_embedding(ids, w, dy)
    assert torch.isnan(dw[40]).all() and torch.isinf(dw[41, 5]) and torch.isfinite(dw[41, :5]).all()
    assert torch.isfinite(dw[:40]).all() and not dw[42:].any()


def test_a_table_beyond_32_bit_offsets():
    g = gen_of("large")
    vocab, n = 140000, 16384  # 2.3e9 values
    w = torch.zeros(vocab, n, dtype=BF16, device=DEV)
    ids = torch.tensor([vocab - 1, 5, vocab - 2, 131073, vocab - 1], device=DEV)
    w[ids] = rnd(g, 5, n, dtype=BF16)
    dy = rnd(g, 5, n, dtype=BF16)
    y, dw = run_embedding(ids, w, dy)
    assert torch.equal(y, w[ids])
    assert torch.equal(dw[5], dy[1]) and torch.equal(dw[vocab - 2], dy[2]) and torch.equal(dw[131073], dy[3])
    assert torch.equal(dw[vocab - 1], (dy[0].float() + dy[4].float()).bfloat16())
    dw[ids] = 0
    assert not dw.any()


# ---- dropout ----------------------------------------------------------------------------------------


def run_dropout(x, p, seed, site, r, dy):
    x = x.detach().requires_grad_(True)
    r = None if r is None else r.detach().requires_grad_(True)
    y = E.dropout(x, p, seed=seed, site=site, residual=r)
    return y.detach(), *torch.autograd.grad(y, (x,) if r is None else (x, r), dy)


def compare_dropout(x, p, seed, site, r, dy, got):
    y, error, kept = R.dropout(x.double(), p, seed, site, None if r is None else r.double(), x.dtype)
    R.check("y", got[0], y, error, x.dtype)
    dx, error, _ = R.dropout(dy.double(), p, seed, site, None, x.dtype)
    R.check("dx", got[1], dx, error, x.dtype)
    if r is not None:
        assert torch.equal(got[2], dy)
    return kept


@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5, 11), (64, 896), (1237, 333), (1500, 1001), (4100, 4099)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_dropouts(dtype, shape):
    g = gen_of(dtype, shape)
    x, r, dy = (rnd(g, *shape, dtype=dtype) for _ in range(3))
    for p, seed, site in ((0.1, 1, 0), (0.5, 2 ** 64 - 3, 5), (0.3, -7, 2 ** 32 - 1), (1e-5, 2 ** 63, 1), (0.999, 0, 3), (0.0, 9, 9), (1.0, 9, 9)):
        for residual in (r, None):
            got = run_dropout(x, p, seed, site, residual, dy)
            compare_dropout(x, p, seed, site, residual, dy, got)


def test_lower_halves_decide_where_upper_ones_tie():
    """A limit whose upper half is met by many values: all but 2^-9 of the numbers that begin with it are dropped."""
    count = 1 << 21
    numbers = R.numbers(count, 77, 4)
    upper = int(numbers[0] >> 16)
    p = (upper * 2 ** 16 + 2 ** 16 - 128) / 2 ** 32
    x, dy = torch.ones(count, device=DEV), torch.ones(count, device=DEV)
    got = run_dropout(x, p, 77, 4, None, dy)
    kept = compare_dropout(x, p, 77, 4, None, dy, got)
    tied = torch.from_numpy((numbers >> 16) == upper).to(DEV)
    assert int(tied.sum()) > 10 and int((tied & ~kept).sum()) > 5


def test_dropped_values_leave_nothing_behind():
    g = gen_of("dropped")
    x = torch.full((4000,), float("nan"), dtype=BF16, device=DEV)
    r = rnd(g, 4000, dtype=BF16)
    y = E.dropout(x, 0.4, seed=3, residual=r)
    kept = torch.isnan(y)
    assert torch.equal(y[~kept], r[~kept]) and 0.55 < kept.float().mean() < 0.65
    dy = torch.full_like(x, float("inf"))
    dx = run_dropout(r, 0.4, 3, 0, None, dy)[1]
    assert torch.equal(dx, torch.where(kept, dy, torch.zeros_like(dy)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_numbers_go_by_the_place_in_a_shape(dtype):
    """Not by strides, addresses, types or what a kernel takes together."""
    g = gen_of("place", dtype)
    x, dy = rnd(g, 90, 50, dtype=dtype), rnd(g, 90, 50, dtype=dtype)
    want = run_dropout(x, 0.25, 11, 2, x, dy)
    for lay in (lambda t: t.t().contiguous().t(), lambda t: torch.cat([t, t], 1)[:, :50], lambda t: torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].view(90, 50),
                lambda t: t.view(9, 10, 50)):
        got = run_dropout(lay(x), 0.25, 11, 2, lay(x), lay(dy))
        assert all(torch.equal(a.reshape(-1), e.reshape(-1)) for a, e in zip(got, want))
    wide = E.dropout(torch.ones(90, 50, device=DEV), 0.25, seed=11, site=2)
    narrow = E.dropout(torch.ones(90, 50, dtype=BF16, device=DEV), 0.25, seed=11, site=2)
    assert torch.equal(wide != 0, narrow != 0)
    assert not torch.equal(wide != 0, E.dropout(torch.ones(90, 50, device=DEV), 0.25, seed=11, site=3) != 0)
    assert not torch.equal(wide != 0, E.dropout(torch.ones(90, 50, device=DEV), 0.25, seed=12, site=2) != 0)


def test_a_seed_in_device_memory():
    g = gen_of("seed")
    x, dy = rnd(g, 70, 33), rnd(g, 70, 33)
    assert torch.equal(E.dropout(x, 0.2, seed=np.int64(5), site=np.int32(1)), E.dropout(x, 0.2, seed=5, site=1))
    for seed in (5, -5, 2 ** 40 + 3):
        at = torch.tensor([seed], device=DEV)
        assert all(torch.equal(a, e) for a, e in zip(run_dropout(x, 0.2, at, 1, x, dy), run_dropout(x, 0.2, seed, 1, x, dy)))
    leaf = x.clone().requires_grad_(True)
    at = torch.tensor(3, device=DEV)
    y = E.dropout(leaf, 0.2, seed=at)
    at += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaf, dy)


def test_shares_that_are_kept():
    """Over n values the share that is dropped lies within 5 standard deviations of p, sites and neighbours are not alike."""
    n = 1 << 22
    ones = torch.ones(n, dtype=BF16, device=DEV)
    for p in (0.01, 0.1, 0.5):
        masks = [E.dropout(ones, p, seed=1234, site=s) == 0 for s in range(2)]
        far = 5 * (p * (1 - p) / n) ** 0.5
        for m in masks:
            assert abs(m.float().mean().item() - p) < far + 2 ** -20
        both, next_to = (masks[0] & masks[1]).float().mean().item(), (masks[0][1:] & masks[0][:-1]).float().mean().item()
        assert abs(both - p * p) < 5 * p / n ** 0.5 and abs(next_to - p * p) < 5 * p / n ** 0.5


# ---- entry points -----------------------------------------------------------------------------------


def test_nothing_is_written_beside_the_results():
    """Results in the middle of larger buffers, at addresses of any element: what lies around them stays as it was."""
    lib, stream = _abi.lib(), torch.cuda.current_stream().cuda_stream
    g = gen_of("beside")
    for dtype in DTYPES:
        code, size = _abi.dtype_code(dtype), dtype.itemsize
        for rows, n in ((5, 77), (33, 264), (3, 5), (2, 4099)):
            count = rows * n

            def around(values):
                return torch.full((values + 14,), 7.0, dtype=dtype, device=DEV)

            def beside(t, values):
                assert bool((t[:7] == 7).all()) and bool((t[7 + values:] == 7).all())

            x, r, dy, ds = (rnd(g, count + 3, dtype=dtype)[3:] for _ in range(4))
            w = rnd(g, n + 1, dtype=dtype)[1:]
            y, s, dx, dw, db = (around(v) for v in (count, count, count, n, n))
            stats = torch.full((2 * rows + 2,), 7.0, device=DEV)
            p = _abi.Norm(kind=_abi.NORM_LAYER, dtype=code, rows=rows, n=n, x=x.data_ptr(), x_row=n, residual=r.data_ptr(), res_row=n, weight=w.data_ptr(), eps=1e-5,
                          y=y.data_ptr() + 7 * size, sum=s.data_ptr() + 7 * size, stats=stats.data_ptr() + 4)
            _abi.check(lib.muon_hip_norm_run(ctypes.addressof(p), stream))
            q = _abi.NormGrad(kind=_abi.NORM_LAYER, dtype=code, rows=rows, n=n, dy=dy.data_ptr(), dy_row=n, s=s.data_ptr() + 7 * size, s_row=n, ds=ds.data_ptr(), ds_row=n,
                              weight=w.data_ptr(), stats=stats.data_ptr() + 4, dx=dx.data_ptr() + 7 * size, dweight=dw.data_ptr() + 7 * size, dbias=db.data_ptr() + 7 * size)
            need = lib.muon_hip_norm_grad_workspace(ctypes.addressof(q))
            ws = torch.full((need + 64,), 9, dtype=torch.uint8, device=DEV)
            assert lib.muon_hip_norm_grad_run(ctypes.addressof(q), ws.data_ptr(), need - 1, stream) == -1
            _abi.check(lib.muon_hip_norm_grad_run(ctypes.addressof(q), ws.data_ptr(), need, stream))
            for t, values in ((y, count), (s, count), (dx, count), (dw, n), (db, n)):
                beside(t, values)
            assert stats[0] == 7 and stats[-1] == 7 and bool((ws[need:] == 9).all())
            got = {"y": y[7:7 + count].view(rows, n), "s": s[7:7 + count].view(rows, n), "dx": dx[7:7 + count].view(rows, n), "dw": dw[7:7 + n], "db": db[7:7 + n]}
            compare_norm("layer", x.view(rows, n), w, None, r.view(rows, n), 1e-5, dy.view(rows, n), ds.view(rows, n), got)

            vocab = 19
            table, out, grad = rnd(g, vocab * n + 1, dtype=dtype)[1:], around(count), around(vocab * n)
            ids = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
            _abi.check(lib.muon_hip_embedding(ids.data_ptr(), 1, rows, table.data_ptr(), n, vocab, n, code, 1.0, out.data_ptr() + 7 * size, stream))
            beside(out, count)
            assert torch.equal(out[7:7 + count].view(rows, n), table.view(vocab, n)[ids])
            need = lib.muon_hip_embedding_grad_workspace(rows, vocab, n, code)
            ws = torch.full((need + 64,), 9, dtype=torch.uint8, device=DEV)
            args = (ids.data_ptr(), 1, rows, dy.data_ptr(), n, vocab, n, code, 1.0, -1, grad.data_ptr() + 7 * size, ws.data_ptr())
            assert lib.muon_hip_embedding_grad(*args, need - 1, stream) == -1
            _abi.check(lib.muon_hip_embedding_grad(*args, need, stream))
            beside(grad, vocab * n)
            assert bool((ws[need:] == 9).all())
            R.check("dw", grad[7:7 + vocab * n].view(vocab, n), *R.embedding_grad(ids, dy.double().view(rows, n), vocab, 1.0), dtype)

            out = around(count)
            _abi.check(lib.muon_hip_dropout(x.data_ptr(), None, out.data_ptr() + 7 * size, count, code, 0.5, 3, None, 1, stream))
            beside(out, count)
            want = E.dropout(x, 0.5, seed=3, site=1)
            assert torch.equal(out[7:7 + count], want)
            own = x.clone()
            _abi.check(lib.muon_hip_dropout(own.data_ptr(), None, own.data_ptr(), count, code, 0.5, 3, None, 1, stream))  # in place
            assert torch.equal(own, want)


# ---- all of them --------------------------------------------------------------------------------------


def test_values_beyond_32_bit_offsets():
    """Tensors of 2.2e9 values: the last rows are those of the same rows alone."""
    rows, n = 262200, 8200
    g = gen_of("far")
    x = torch.zeros(rows, n, dtype=BF16, device=DEV)
    tail, w = rnd(g, 24, n, dtype=BF16), rnd(g, n, dtype=BF16)
    x[-24:] = tail
    y, s = E.rms_norm(x, w, residual=x)
    want = E.rms_norm(tail, w, residual=tail)
    # (a row's sums may have another order where there are many rows)
    R.check("y", y[-24:], want[0].double(), 1e-5 * want[0].double().abs() + R.unit(BF16) * want[0].double().abs(), BF16)
    assert torch.equal(s[-24:], want[1]) and not s[:-24].any()
    del y, s
    y = E.dropout(x, 0.3, seed=8)[-24:].clone()
    first = (rows - 24) * n
    assert first % 8 == 0 and first > 2 ** 31
    kept = torch.from_numpy(R.numbers(24 * n, 8, 0, first) >= int(np.rint(0.3 * 2 ** 32))).to(DEV).view(24, n)
    assert torch.equal(y != 0, kept & (tail != 0))


def everything(x, ids, table, w, b, seed):
    """All four, forward and backward, from one leaf to one loss."""
    e = E.embedding(ids, table, scale=2.0)
    h = E.dropout(e, 0.1, seed=seed, site=0, residual=x)
    y, s = E.layer_norm(h, w, b, residual=e)
    z, s = E.rms_norm(E.dropout(y, 0.2, seed=seed, site=1), w, residual=s)
    return (z.float() * z.float()).sum() + s.float().sum()


def leaves_of(g, dtype, t=50, n=264, v=31):
    x, table, w, b = (rnd(g, *shape, dtype=dtype).requires_grad_(True) for shape in ((t, n), (v, n), (n,), (n,)))
    return x, torch.randint(0, v, (t,), generator=g, device=DEV), table, w, b


@pytest.mark.parametrize("dtype", DTYPES)
def test_passes_are_recorded_and_replayed(dtype):
    """A training pass in a graph draws other numbers at every replay, where the seed is one of its tensors."""
    g = gen_of("graph", dtype)
    x, ids, table, w, b = leaves_of(g, dtype)
    leaves = (x, table, w, b)
    seed = torch.tensor([100], device=DEV)

    def step():
        grads = torch.autograd.grad(everything(x, ids, table, w, b, seed), leaves)
        seed.add_(1)
        return grads

    want = [step() for _ in range(4)]
    assert not torch.equal(want[0][0], want[1][0])
    seed.fill_(100)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    seed.fill_(100)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(got, want[i]):
            assert torch.equal(a, e), i
        if i == 1:
            everything(x.detach(), ids, table.detach(), w.detach(), b.detach(), 5)  # eager work of the program's own in between


def test_two_graphs_take_turns():
    """Each has workspaces of its own, whichever is replayed between two replays of the other."""
    g = gen_of("two graphs")
    sets = [leaves_of(g, BF16, t=t, n=264, v=77) for t in (50, 700)]

    def grads(i):
        x, ids, table, w, b = sets[i]
        return torch.autograd.grad(everything(x, ids, table, w, b, 3 + i), (x, table, w, b))

    want = [grads(i) for i in range(2)]
    torch.cuda.synchronize()
    graphs, got = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            got.append(grads(i))
    for i in (0, 1, 1, 0, 1, 0):
        for t in got[i]:
            t.zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(got[i], want[i])), i


def test_two_streams_at_once():
    g = gen_of("streams")
    sets = [leaves_of(g, BF16, t=600, n=1000, v=200) for _ in range(2)]

    def grads(i):
        x, ids, table, w, b = sets[i]
        return torch.autograd.grad(everything(x, ids, table, w, b, i), (x, table, w, b))

    want = [grads(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            got.append([grads(i) for _ in range(5)])
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i]:
            assert all(torch.equal(a, e) for a, e in zip(one, want[i]))


@pytest.mark.parametrize("name,call", [("embedding", lambda x, w: E.embedding(torch.arange(3, device=DEV), x)), ("layer_norm", lambda x, w: E.layer_norm(x, w, w)),
                                       ("rms_norm", lambda x, w: E.rms_norm(x, w)), ("dropout", lambda x, w: E.dropout(x, 0.5, seed=1))])
def test_what_is_not_differentiated_raises(name, call):
    g = gen_of(name)
    x, w = rnd(g, 4, 16).requires_grad_(True), rnd(g, 16).requires_grad_(True)
    y = call(x, w)
    dy = torch.ones_like(y).requires_grad_(True)
    (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(dx.sum(), dy)
    if "norm" in name:
        with pytest.raises(RuntimeError, match="differentiated once"):
            torch.autograd.grad(torch.autograd.grad(call(x, w), x, torch.ones_like(y), create_graph=True)[0].sum(), x)
        with pytest.raises(RuntimeError, match="differentiated once"):
            torch.autograd.grad(torch.autograd.grad(call(x, w), w, torch.ones_like(y), create_graph=True)[0].sum(), x)
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level(), pytest.raises(RuntimeError):
        call(fwAD.make_dual(x.detach(), torch.ones_like(x)), w)


def test_inputs_that_gradients_read_may_not_change():
    g = gen_of("changed")
    x, w = rnd(g, 4, 16).requires_grad_(True), rnd(g, 16).requires_grad_(True)
    r = rnd(g, 4, 16)
    y, s = E.rms_norm(x, w, residual=r)
    r.zero_()  # nothing reads it again
    torch.autograd.grad(y.sum(), (x, w), retain_graph=True)
    with torch.no_grad():
        s.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), (x, w))
    ids = torch.arange(4, device=DEV)
    y = E.embedding(ids, x)
    ids.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)


CALLS = {"embedding": lambda x, w: E.embedding(torch.arange(3, device=DEV), x), "layer_norm": lambda x, w: E.layer_norm(x, w, residual=x)[0],
         "rms_norm": lambda x, w: E.rms_norm(x, w), "dropout": lambda x, w: E.dropout(x, 0.5, seed=1, residual=x)}


def both_ways(f, x, w):
    y = f(x, w)
    leaves = [t for t in (x, w) if t.requires_grad]
    return [y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y), allow_unused=True)]


@pytest.mark.parametrize("record", RECORDERS)
@pytest.mark.parametrize("name", list(CALLS))
def test_recording_is_refused(name, record):
    x, w = torch.ones(4, 16, device=DEV), torch.ones(16, device=DEV)
    with pytest.raises(NotImplementedError, match="recorded"):
        record(CALLS[name], x, w)
    y = CALLS[name](x.requires_grad_(True), w)
    with pytest.raises(NotImplementedError, match="recorded"):
        make_fx(lambda dy: torch.autograd.grad(y, x, dy, retain_graph=True)[0])(torch.ones_like(y))
    assert torch.isfinite(torch.autograd.grad(y, x, torch.ones_like(y))[0]).all()  # and afterwards calls are taken again


@pytest.mark.parametrize("name", list(CALLS))
def test_recomputed_and_compiled_passes_give_the_same(name):
    from torch.utils.checkpoint import checkpoint
    from torch.utils.flop_counter import FlopCounterMode

    g = gen_of(name, "again")
    x, w = rnd(g, 6, 16).requires_grad_(True), rnd(g, 16).requires_grad_(True)

    def f(a, b):
        return CALLS[name](a * 2, b).relu() + 1

    def same(got):
        for a, e in zip(got, both_ways(f, x, w)):
            assert a is e is None or torch.equal(a, e)

    same(both_ways(lambda a, b: checkpoint(f, a, b, use_reentrant=False), x, w))
    same(both_ways(torch.compile(f, backend="eager"), x, w))
    with FlopCounterMode(display=False):
        got = both_ways(f, x, w)
    same(got)


@pytest.mark.parametrize("name", list(CALLS))
def test_the_same_tensor_twice_and_parameters(name):
    """A tensor that is input and residual at once gets both gradients; parameters are tensors like others."""
    g = gen_of(name, "twice")
    x, r, w = rnd(g, 5, 40), rnd(g, 5, 40), rnd(g, 40)
    if name == "embedding":
        p = torch.nn.Parameter(x)
        ids = torch.tensor([1, 1, 4], device=DEV)
        (E.embedding(ids, p).sum() + E.embedding(ids, p, scale=2.0).sum()).backward()
        assert torch.equal(p.grad.sum(1), torch.tensor([0.0, 240.0, 0.0, 0.0, 120.0], device=DEV))
        return
    call = {"layer_norm": lambda a, b: E.layer_norm(a, w, residual=b), "rms_norm": lambda a, b: E.rms_norm(a, w, residual=b),
            "dropout": lambda a, b: (E.dropout(a, 0.5, seed=1, residual=b),)}[name]
    p = torch.nn.Parameter(x)
    outs = call(p, p)
    torch.autograd.backward(outs, [torch.ones_like(o) for o in outs])
    a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    outs = call(a, b)
    torch.autograd.backward(outs, [torch.ones_like(o) for o in outs])
    assert torch.equal(p.grad, a.grad + b.grad)
    a.grad.zero_()  # each leaf has a gradient of its own
    assert b.grad.any()


def test_results_under_inference_mode():
    g = gen_of("inference")
    x, w = rnd(g, 6, 48, dtype=BF16), rnd(g, 48, dtype=BF16)
    ids = torch.tensor([5, 0], device=DEV)
    want = [E.layer_norm(x, w, w), *E.rms_norm(x, w, residual=x), E.dropout(x, 0.5, seed=1), E.embedding(ids, x)]
    with torch.inference_mode():
        got = [E.layer_norm(x, w, w), *E.rms_norm(x, w, residual=x), E.dropout(x, 0.5, seed=1), E.embedding(ids, x)]
        assert all(t.is_inference() for t in got)
        again = E.rms_norm(got[0], w)
    assert all(torch.equal(a, e) for a, e in zip(got, want)) and torch.equal(again, E.rms_norm(want[0], w))
    assert not any(t.is_inference() for t in want)


def test_kernels_are_timed_by_name():
    x = torch.ones(4, 64, device=DEV)
    _abi.timing_enable(True)
    try:
        E.rms_norm(x)
        E.dropout(x, 0.5, seed=1)
        E.embedding(torch.arange(3, device=DEV), x)
        seen = _abi.timing_read()
    finally:
        _abi.timing_enable(False)
    assert all(seen[k][1] == 1 for k in ("norm", "dropout", "embedding"))
