"""linear and gated_linear against their formulas in 64 bits: results and every gradient, at the sizes, layouts and values where tiles,
reductions and masks can go wrong.  Bounds: tests/layer_reference.py."""
import ctypes
import itertools

import pytest
import torch

import lmms_engine_amd as E
from lmms_engine_amd import _abi, layers
from lmms_engine_amd.clip_grad import clip_grad_norm_
from tests import layer_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F = torch.bfloat16, torch.float32


def rnd(gen, *shape, scale=1.0, dtype=BF):
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


def gen_of(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def run_linear(x, w, b, r, name, dy):
    leaves = [t for t in (x, w, b, r) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y = E.linear(x, w, b, activation=name, residual=r)
    grads = iter(torch.autograd.grad(y, leaves, dy))
    got = {"y": y, "dx": next(grads), "dw": next(grads)}
    if b is not None:
        got["db"] = next(grads)
    if r is not None:
        got["dr"] = next(grads)
    with torch.no_grad():  # the call that keeps nothing gives the same bits
        assert torch.equal(E.linear(x, w, b, activation=name, residual=r).view(torch.uint8), y.detach().view(torch.uint8))
    return got


def run_gated(x, wg, wu, bg, bu, name, dh):
    leaves = [t for t in (x, wg, wu, bg, bu) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y = E.gated_linear(x, wg, wu, bg, bu, activation=name)
    names = ["dx", "dw0", "dw1"] + (["db0"] if bg is not None else []) + (["db1"] if bu is not None else [])
    got = {"y": y, **dict(zip(names, torch.autograd.grad(y, leaves, dh)))}
    with torch.no_grad():
        assert torch.equal(E.gated_linear(x, wg, wu, bg, bu, activation=name).view(torch.uint8), y.detach().view(torch.uint8))
    return got


def compare(got, want):
    for name, value in got.items():
        R.check(name, value.reshape(want[name][0].shape), *want[name])


# tokens, inner, outer: single values and rows, the edges of pieces, fragments, tiles and k-tiles, long reductions over few results
SIZES = [(1, 1, 1), (1, 64, 8), (3, 8, 5), (2, 7, 64), (16, 64, 64), (17, 251, 33), (64, 128, 64), (65, 130, 129), (130, 72, 264), (33, 1000, 77),
         (257, 96, 520), (1, 4096, 512), (5, 2049, 130), (2000, 24, 40), (700, 200, 1000), (8, 250, 35),
         (9, 250, 35), (6, 4100, 17), (40, 9000, 24)]
ACTS = list(layers.ACTIVATIONS)


@pytest.mark.parametrize("dtype", [BF, F], ids=["bf16", "f32"])
@pytest.mark.parametrize("i,size", list(enumerate(SIZES)), ids=["x".join(map(str, s)) for s in SIZES])
def test_linear(dtype, i, size):
    t, k, n = size
    g = gen_of(i)
    name, bias, residual = ACTS[i % 6], i % 2 == 0, i % 3 != 0
    x, w = rnd(g, t, k, dtype=dtype), rnd(g, n, k, scale=k ** -0.5, dtype=dtype)
    b = rnd(g, n, dtype=dtype) if bias else None
    r = rnd(g, t, n, dtype=dtype) if residual else None
    dy = rnd(g, t, n, dtype=dtype)
    compare(run_linear(x, w, b, r, name, dy), R.linear(x, w, b, r, name, dy, dtype))


@pytest.mark.parametrize("dtype", [BF, F], ids=["bf16", "f32"])
@pytest.mark.parametrize("i,size", list(enumerate(SIZES)), ids=["x".join(map(str, s)) for s in SIZES])
def test_gated_linear(dtype, i, size):
    t, k, n = size
    g = gen_of(100 + i)
    name = ACTS[(i + 3) % 6]
    x = rnd(g, t, k, dtype=dtype)
    wg, wu = (rnd(g, n, k, scale=k ** -0.5, dtype=dtype) for _ in range(2))
    bg, bu = (rnd(g, n, dtype=dtype) if i % 4 in wanted else None for wanted in ((1, 3), (2, 3)))
    dh = rnd(g, t, n, dtype=dtype)
    compare(run_gated(x, wg, wu, bg, bu, name, dh), R.gated(x, wg, wu, bg, bu, name, dh, dtype))


@pytest.mark.parametrize("dtype", [BF, F], ids=["bf16", "f32"])
@pytest.mark.parametrize("steps", range(1, 30))
def test_few_rows_with_every_rest(dtype, steps):
    """Up to eight rows, whose reduction eight waves share in batches of fragments: every number of fragments that may be left for a wave."""
    g = gen_of(300 + steps)
    step = 32 if dtype == BF else 16
    for k in (8 * step * steps, 8 * step * steps - 3 * step - 5):
        x, w, w2 = rnd(g, 1 + steps % (8, 4)[steps % 2], k, dtype=dtype), *(rnd(g, 40, k, scale=k ** -0.5, dtype=dtype) for _ in range(2))
        dy = torch.zeros(x.size(0), 40, dtype=dtype, device=DEV)
        for _ in range(2):
            R.check("linear", E.linear(x, w), *R.linear(x, w, None, None, "none", dy, dtype)["y"])
            R.check("gated", E.gated_linear(x, w, w2), *R.gated(x, w, w2, None, None, "silu", dy, dtype)["y"])


# Results of many tiles: every tile size, also for gradients, whole and ragged in every direction.
LARGE = [(2060, 200, 2056), (4100, 136, 4200), (136, 4100, 4200), (4100, 4200, 72), (4352, 320, 4096), (1024, 1024, 1024), (4099, 100, 4103)]


@pytest.mark.parametrize("dtype", [BF, F], ids=["bf16", "f32"])
@pytest.mark.parametrize("i,size", list(enumerate(LARGE)), ids=["x".join(map(str, s)) for s in LARGE])
def test_many_tiles(dtype, i, size):
    t, k, n = size
    g = gen_of(200 + i)
    x, w, w2, b = rnd(g, t, k, dtype=dtype), *(rnd(g, n, k, scale=k ** -0.5, dtype=dtype) for _ in range(2)), rnd(g, n, dtype=dtype)
    r, dy = rnd(g, t, n, dtype=dtype), rnd(g, t, n, dtype=dtype)
    name = ("gelu", "none")[i % 2]
    compare(run_linear(x, w, b, r, name, dy), R.linear(x, w, b, r, name, dy, dtype))
    compare(run_gated(x, w, w2, None, b, "silu", dy), R.gated(x, w, w2, None, b, "silu", dy, dtype))


@pytest.mark.parametrize("dtype", [BF, F], ids=["bf16", "f32"])
@pytest.mark.parametrize("name", ACTS)
def test_activations_from_end_to_end(dtype, name):
    """Every activation over its whole range, subnormal and huge arguments included: z = x * 1 is the argument itself."""
    v = torch.cat([torch.linspace(-30, 30, 1501), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e-39, 88.8, -88.8, 200.0, -200.0, 1e4, -1e4, 1e18, -1e18])])
    x = v.to(dtype).to(DEV)[:, None]
    one = torch.ones(1, 1, dtype=dtype, device=DEV)
    dy = torch.ones_like(x)
    compare(run_linear(x, one, None, None, name, dy), R.linear(x, one, None, None, name, dy, dtype))
    compare(run_gated(x, one, one.detach().clone(), None, None, name, dy), R.gated(x, one, one, None, None, name, dy, dtype))


@pytest.mark.parametrize("size", [(0, 8, 4), (5, 0, 7), (4, 8, 0), (0, 0, 0), (0, 5, 3)], ids=str)
def test_empty_sizes(size):
    t, k, n = size
    g = gen_of(7)
    x, w, b, r, dy = rnd(g, t, k), rnd(g, n, k), rnd(g, n), rnd(g, t, n), rnd(g, t, n)
    compare(run_linear(x, w, b, r, "silu", dy), R.linear(x, w, b, r, "silu", dy, BF))
    compare(run_gated(x, w, w.detach().clone(), b, b.detach().clone(), "gelu", dy), R.gated(x, w, w, b, b, "gelu", dy, BF))


def layouts(g, rows, cols, dtype):
    """The same kind of matrix in the layouts that callers have; what lies around it is NaN."""
    def inside(shape, cut):
        buf = torch.full(shape, float("nan"), dtype=dtype, device=DEV)
        view = cut(buf)
        view.copy_(rnd(g, *view.shape, dtype=dtype))
        return view

    yield "transposed", inside((cols, rows), lambda b: b.t())
    yield "wide rows", inside((rows, cols + 16), lambda b: b[:, 8:8 + cols])
    yield "odd offset", inside((rows, cols + 3), lambda b: b[:, 1:1 + cols])
    yield "transposed of wide rows", inside((cols, rows + 24), lambda b: b[:, 16:16 + rows].t())
    yield "every other", inside((rows, 2 * cols), lambda b: b[:, ::2])
    yield "aligned rows of odd length", inside((rows, -(-cols // 8) * 8 + 8), lambda b: b[:, :cols])
    yield "one row for all", rnd(g, 1, cols, dtype=dtype).expand(rows, cols)
    yield "one value per row", rnd(g, rows, 1, dtype=dtype).expand(rows, cols)


LAYOUTS = ["transposed", "wide rows", "odd offset", "transposed of wide rows", "every other", "aligned rows of odd length", "one row for all",
           "one value per row"]


@pytest.mark.parametrize("dtype", [BF, F], ids=["bf16", "f32"])
@pytest.mark.parametrize("size", [(72, 136, 200), (45, 99, 70)], ids=str)
@pytest.mark.parametrize("which", ["x", "w", "r", "dy"])
def test_layouts(which, size, dtype):
    t, k, n = size
    shape = dict(x=(t, k), w=(n, k), r=(t, n), dy=(t, n))[which]
    for i, (name, view) in enumerate(layouts(gen_of(3), *shape, dtype)):
        assert name == LAYOUTS[i]
        g = gen_of(50 + i)
        v = dict(x=rnd(g, t, k, dtype=dtype), w=rnd(g, n, k, scale=k ** -0.5, dtype=dtype), r=rnd(g, t, n, dtype=dtype), dy=rnd(g, t, n, dtype=dtype))
        v[which] = view.detach()
        for act in ("none", "silu"):
            compare(run_linear(v["x"].detach(), v["w"].detach(), None, v["r"].detach(), act, v["dy"]), R.linear(v["x"], v["w"], None, v["r"], act, v["dy"], dtype))
        if which == "r":
            continue
        other = rnd(g, n, k, scale=k ** -0.5, dtype=dtype)
        for wg, wu in ((v["w"], other), (other, v["w"])):
            compare(run_gated(v["x"].detach(), wg.detach(), wu.detach(), None, None, "silu", v["dy"]),
                    R.gated(v["x"], wg, wu, None, None, "silu", v["dy"], dtype))


def test_leading_dimensions():
    g = gen_of(9)
    x, w, r = rnd(g, 3, 5, 40), rnd(g, 24, 40, scale=0.2), rnd(g, 3, 5, 24)
    y = E.linear(x, w, residual=r)
    assert y.shape == (3, 5, 24) and torch.equal(y.view(15, 24), E.linear(x.view(15, 40), w, residual=r.view(15, 24)))
    t = x.transpose(0, 1)
    assert torch.equal(E.linear(t, w), E.linear(t.contiguous(), w))
    one = E.linear(x[0, 0], w)
    assert one.shape == (24,) and torch.equal(one, E.linear(x, w)[0, 0])
    assert E.gated_linear(x[1, 2], w, w).shape == (24,)
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(E.linear(x.transpose(0, 1), w).float().sum(), x)
    assert dx.shape == x.shape


def test_values_that_are_not_finite_stay_in_their_rows():
    """A NaN or an infinity of x or W reaches the results that contain it and no other; so do gradients."""
    g = gen_of(11)
    t, k, n = 140, 200, 150
    x, w, dy = rnd(g, t, k), rnd(g, n, k, scale=0.1), rnd(g, t, n)
    clean = E.linear(x, w)
    x[7, 3], x[131, 199], w[149, 0] = float("nan"), float("inf"), float("-inf")
    y = E.linear(x, w)
    want = x.double() @ w.double().t()
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want))
    keep = torch.isfinite(want)
    assert torch.equal(y[keep], clean[keep])
    dy[3, 5] = float("nan")
    dx, dw = torch.autograd.grad(E.linear(x.requires_grad_(True), w.requires_grad_(True)), (x, w), dy)
    assert torch.isnan(dx[3]).all() and torch.isfinite(dx[4, 1:]).all()
    assert torch.isnan(dw[5]).all() and torch.isfinite(dw[6, :3]).all() and torch.isnan(dw[6, 3]) and not torch.isfinite(dw[6, 199])


def test_each_gradient_alone():
    """What is not asked for is not computed, and what is asked for does not depend on what else is."""
    g = gen_of(13)
    t, k, n = 50, 72, 88
    make = dict(x=rnd(g, t, k), wg=rnd(g, n, k, scale=0.2), wu=rnd(g, n, k, scale=0.2), bg=rnd(g, n), bu=rnd(g, n))
    dh = rnd(g, t, n)

    def grads(names):
        v = {m: a.clone().requires_grad_(m in names) for m, a in make.items()}
        y = E.gated_linear(v["x"], v["wg"], v["wu"], v["bg"], v["bu"])
        return dict(zip(names, torch.autograd.grad(y, [v[m] for m in names], dh)))

    whole = grads(list(make))
    for some in itertools.chain(itertools.combinations(make, 1), itertools.combinations(make, 2)):
        for m, a in grads(list(some)).items():
            assert torch.equal(a, whole[m]), (some, m)
    lin = dict(x=make["x"], w=make["wg"], b=make["bg"], r=rnd(g, t, n))

    def lgrads(names, act):
        v = {m: a.clone().requires_grad_(m in names) for m, a in lin.items()}
        return dict(zip(names, torch.autograd.grad(E.linear(v["x"], v["w"], v["b"], activation=act, residual=v["r"]), [v[m] for m in names], dh)))

    for act in ("none", "gelu"):
        whole = lgrads(list(lin), act)
        for some in itertools.combinations(lin, 1):
            for m, a in lgrads(list(some), act).items():
                assert torch.equal(a, whole[m]), (act, m)


def test_gradients_against_differences():
    """The gradients of a scalar against central differences of the function itself, in fp32: a step of 2^-6 along a random direction.
    The differences are off by the third derivative (a sixth of the step squared times it) and by the rounding of two sums."""
    g = gen_of(17)
    t, k, n = 12, 40, 24
    for name in ("sigmoid", "silu", "gelu", "gelu_tanh"):
        v = [rnd(g, t, k, dtype=F), rnd(g, n, k, scale=0.15, dtype=F), rnd(g, n, k, scale=0.15, dtype=F), rnd(g, n, dtype=F), rnd(g, n, dtype=F)]
        c = rnd(g, t, n, dtype=F).double()
        for f in (lambda a: E.gated_linear(*a, activation=name), lambda a: E.linear(a[0], a[1], a[3], activation=name)):
            leaves = [a.clone().requires_grad_(True) for a in v]
            grads = torch.autograd.grad(f(leaves), leaves, c.float(), allow_unused=True)
            for i, gi in enumerate(grads):
                if gi is None:
                    continue
                d = rnd(g, *v[i].shape, dtype=F)
                d /= d.norm()
                h = 2.0 ** -6
                with torch.no_grad():
                    up, down = (f([a + s * h * d if j == i else a for j, a in enumerate(v)]).double() for s in (1, -1))
                slope = ((up - down) * c).sum().item() / (2 * h)
                told = (gi.double() * d.double()).sum().item()
                # |x| <= 6, |w| <= 1: a direction of norm 1 moves z by at most 7, third derivatives of the factors stay below 2 * 7^3 * max(1, |u|)
                room = (h * h / 6 * 2 * 7 ** 3 * 8 * c.abs().mean().item() + 2 ** -22 * 8 * c.abs().sum().item() / h)
                assert abs(slope - told) <= room, (name, i, slope, told, room)


def product(kind, x, m, n, k, a, b, out):
    """One muon_hip_product_run on row-major operands."""
    lib = _abi.lib()
    p = _abi.Product(kind=kind, dtype=_abi.dtype_code(x.dtype), m=m, n=n, k=k)
    for field, pair in (("a", a), ("b", b)):
        getattr(p, field)[:] = [t.data_ptr() for t in pair]
        getattr(p, field + "_row")[:] = [t.stride(0) for t in pair]
        getattr(p, field + "_col")[:] = [t.stride(1) for t in pair]
    p.out[:] = [t.data_ptr() for t in out]
    need = lib.muon_hip_product_workspace(ctypes.addressof(p))
    assert need >= 0
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
    _abi.check(lib.muon_hip_product_run(ctypes.addressof(p), ws.data_ptr(), need, _abi.stream_ptr(x.device)), "product")


def test_rows_behind_the_result_are_left_alone():
    """Results at the end of a tile that reaches past them: what lies around them in memory stays as it was."""
    g = gen_of(19)
    for (t, k, n), kind in itertools.product([(5, 64, 24), (70, 64, 72), (130, 520, 9)], (_abi.PRODUCT_LINEAR, _abi.PRODUCT_GATED, _abi.PRODUCT_EACH)):
        x, x2, w, w2 = rnd(g, t, k), rnd(g, t, k), rnd(g, n, k), rnd(g, n, k)
        bufs = [torch.full((t * n + 4096,), 7.0, dtype=BF, device=DEV) for _ in range(2)]
        out = [b[2048:2048 + t * n].view(t, n) for b in bufs]
        product(kind, x, t, n, k, (x, x2), (w, w2), out)
        for o, b, left in zip(out, bufs, (x, x2)):
            assert (b[:2048] == 7).all() and (b[2048 + t * n:] == 7).all()
            if kind == _abi.PRODUCT_EACH:
                assert torch.equal(o, E.linear(left, w))
        if kind != _abi.PRODUCT_EACH:
            assert (bufs[1] == 7).all()
            assert torch.equal(out[0], E.linear(x, w) if kind == _abi.PRODUCT_LINEAR else E.gated_linear(x, w, w2, activation="none"))


def test_results_past_four_gib():
    """Rows whose elements are more than 2^32 bytes from the first."""
    t, k, n = 2 ** 17 + 3, 64, 20000
    g = gen_of(23)
    x, w = rnd(g, t, k), rnd(g, n, k, scale=0.1)
    y = E.linear(x, w)
    assert y.numel() > 2 ** 31
    for rows in (slice(0, 40), slice(t // 2, t // 2 + 40), slice(t - 40, t)):
        want = R.linear(x[rows], w, None, None, "none", torch.zeros(40, n, device=DEV), BF)
        R.check("y", y[rows], *want["y"])
    # and as an operand: the gradient of x reads all of it
    dx = E.linear(y, w.t())
    rows = slice(t - 40, t)
    R.check("dx", dx[rows], *R.linear(y[rows], w.t(), None, None, "none", torch.zeros(40, k, device=DEV), BF)["y"])


def block(x, p):
    """A feed-forward block with its residual."""
    return E.linear(E.gated_linear(x, p["gate"], p["up"]), p["down"], residual=x)


def block_by_torch(x, p):
    v = torch.nn.functional
    return x + v.linear(v.silu(v.linear(x, p["gate"])) * v.linear(x, p["up"]), p["down"])


def test_a_block_is_trained_by_the_step():
    """The operators as a training loop uses them: forward, loss gradient, backward into .grad, clipping, Muon step.  The gradients are those of
    the block in 64 bits; what the step makes of them is what it makes of the same gradients without the operators."""
    g = gen_of(29)
    d, inter, t = 128, 320, 200
    init = {"gate": rnd(g, inter, d, scale=d ** -0.5), "up": rnd(g, inter, d, scale=d ** -0.5), "down": rnd(g, d, inter, scale=inter ** -0.5)}
    mine = {m: torch.nn.Parameter(a.clone()) for m, a in init.items()}
    twin = {m: torch.nn.Parameter(a.clone()) for m, a in init.items()}
    opts = [E.Muon([dict(params=list(p.values()), use_muon=True, lr=0.02, rms_scale=False)]) for p in (mine, twin)]
    for step in range(3):
        x, dy = rnd(g, 4, t // 4, d), rnd(g, 4, t // 4, d, scale=1e-2)
        y = block(x, mine)
        y.backward(dy)
        wide = {m: a.detach().double().requires_grad_(True) for m, a in mine.items()}
        grads = torch.autograd.grad(block_by_torch(x.double(), wide), list(wide.values()), dy.double())
        for (m, p), want, (_, q) in zip(mine.items(), grads, twin.items()):
            # h, its factors and two gradients are rounded to bf16 on the way (each 2^-8 of its own size at most, so less of a sum's norm)
            err = ((p.grad.double() - want).norm() / want.norm()).item()
            assert err <= 5 * 2.0 ** -8, (step, m, err)
            q.grad = p.grad.clone()
        for params, opt in zip((mine, twin), opts):
            clip_grad_norm_(params.values(), 1.0)
            opt.step()
            opt.zero_grad(set_to_none=True)
        for m in mine:
            assert torch.equal(mine[m], twin[m])
            assert not torch.equal(mine[m], init[m])


def test_forward_and_backward_in_a_graph():
    """Recorded once, replayed with other inputs in the same memory, with eager calls and synchronizations between."""
    g = gen_of(31)
    t, k, n = 96, 256, 200
    x, dy = rnd(g, t, k).requires_grad_(True), rnd(g, t, n)
    w = [rnd(g, n, k, scale=0.1).requires_grad_(True) for _ in range(2)]
    b = rnd(g, n).requires_grad_(True)

    def both():
        h = E.gated_linear(x, w[0], w[1], b, None)
        y = E.linear(x, w[0], b, activation="gelu", residual=h)
        return [y.detach(), *torch.autograd.grad(y, [x, *w, b], dy)]  # (no history outlives the call)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for r in range(4):
        with torch.no_grad():
            x.copy_(rnd(g, t, k))
            dy.copy_(rnd(g, t, n))
            b.copy_(rnd(g, n))
        graph.replay()
        torch.cuda.synchronize()
        now = [a.detach().clone() for a in held]
        for a, e in zip(now, both()):
            assert torch.equal(a, e.detach()), r


def test_two_streams_at_once():
    """Calls on two streams share nothing: each gives what it gives alone."""
    g = gen_of(37)
    x, w = rnd(g, 48, 4096), rnd(g, 520, 4096, scale=0.02)
    x2, w2 = rnd(g, 40, 4096), rnd(g, 520, 4096, scale=0.02)
    want, want2 = E.linear(x, w, activation="silu"), E.gated_linear(x2, w, w2)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    got, got2 = [], []
    for _ in range(8):
        with torch.cuda.stream(s1):
            got.append(E.linear(x, w, activation="silu"))
        with torch.cuda.stream(s2):
            got2.append(E.gated_linear(x2, w, w2))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) for a in got) and all(torch.equal(a, want2) for a in got2)


def test_the_same_call_gives_the_same_bits():
    g = gen_of(41)
    x, w, dy = rnd(g, 300, 2000), rnd(g, 264, 2000, scale=0.02), rnd(g, 300, 264)
    first = run_linear(x, w, None, None, "silu", dy)
    for _ in range(3):
        for m, a in run_linear(x, w, None, None, "silu", dy).items():
            assert torch.equal(a, first[m]), m


def test_a_second_derivative_raises():
    """The backward pass has none of its own; the residual's, which is the incoming gradient itself, has."""
    g = gen_of(43)
    x, w, r = rnd(g, 8, 16).requires_grad_(True), rnd(g, 24, 16).requires_grad_(True), rnd(g, 8, 24).requires_grad_(True)
    for y in (E.linear(x, w, activation="silu"), E.gated_linear(x, w, w)):
        (dx,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated once"):
            dx.float().sum().backward()
    (dr,) = torch.autograd.grad(E.linear(x, w, residual=r).float().square().sum(), r, create_graph=True)
    dr.float().sum().backward()


def test_forward_mode_is_refused():
    """A tangent is not dropped silently."""
    x, w = rnd(gen_of(67), 4, 16, dtype=F), rnd(gen_of(68), 8, 16, dtype=F)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for f in (lambda: E.linear(dual, w), lambda: E.gated_linear(dual, w, w), lambda: E.linear(x, w, residual=torch.autograd.forward_ad.make_dual(rnd(gen_of(69), 4, 8, dtype=F), torch.ones(4, 8, device=DEV)))):
            with pytest.raises(RuntimeError):
                f()


def test_leaves_that_are_used_twice():
    """x as its own weight, and one weight for both factors: both contributions arrive."""
    g = gen_of(71)
    x = rnd(g, 24, 24, dtype=F).requires_grad_(True)
    (got,) = torch.autograd.grad(E.linear(x, x).square().sum(), x)
    y = x.detach().double().requires_grad_(True)
    (want,) = torch.autograd.grad((y @ y.t()).square().sum(), y)
    assert ((got - want).norm() / want.norm()).item() <= 64 * R.F32 * 24 ** 0.5
    w = rnd(g, 16, 24, dtype=F, scale=0.2).requires_grad_(True)
    (got,) = torch.autograd.grad(E.gated_linear(x.detach(), w, w, activation="sigmoid").sum(), w)
    v = w.detach().double().requires_grad_(True)
    z = x.detach().double() @ v.t()
    (want,) = torch.autograd.grad((torch.sigmoid(z) * z).sum(), v)
    assert ((got - want).norm() / want.norm()).item() <= 64 * R.F32 * 24 ** 0.5


def test_what_the_entry_points_refuse_is_raised_as_the_packages_error():
    """Rows of which a tile spans more than 31 bits reach, forward; the same in a backward pass, which runs on a thread of its own."""
    long = torch.zeros(41, 30_000_001, dtype=BF, device=DEV)
    with pytest.raises(_abi.MuonHipError, match="2 GiB"):
        E.linear(long[:, 1:], torch.zeros(3, 30_000_000, dtype=BF, device=DEV))
    del long
    x, w = torch.ones(300, 1, dtype=BF, device=DEV, requires_grad=True), torch.ones(4_300_000, 1, dtype=BF, device=DEV)
    y = E.linear(x, w)
    assert (y == 1).all()
    with pytest.raises(_abi.MuonHipError, match="2 GiB"):
        torch.autograd.grad(y, x, y.detach())


def test_more_tokens_than_a_row_may_span():
    """The reduction of a weight's gradient over millions of rows that have to be copied first.  Whole numbers: every partial sum is exact."""
    g = gen_of(53)
    t, k, n = 4_400_003, 9, 5
    x = torch.randint(-1, 2, (t, k), generator=g, device=DEV).to(BF)
    dy = torch.randint(-1, 2, (t, n), generator=g, device=DEV).to(BF)
    w, b = torch.zeros(n, k, dtype=F, device=DEV), torch.zeros(n, dtype=F, device=DEV)
    for dt in (F, BF):
        xs, ws, bs = x.to(dt), w.to(dt).requires_grad_(True), b.to(dt).requires_grad_(True)
        dw, db = torch.autograd.grad(E.linear(xs, ws, bs), (ws, bs), dy.to(dt))
        want = dy.double().t() @ x.double()
        assert want.abs().max() < 2 ** 24
        assert torch.equal(dw.double(), want.to(dt).double()) and torch.equal(db.double(), dy.double().sum(0).to(dt).double())


def test_activation_gradients_leave_the_room_between_rows():
    """muon_hip_act_grad on rows further apart than they are long, with two factors, one or none, and with sums or results alone."""
    lib, g = _abi.lib(), gen_of(59)
    for dtype, (m, n) in itertools.product((BF, F), ((5, 7), (70, 264), (600, 1001))):
        dy, one = rnd(g, m, n, dtype=dtype), torch.ones(1, 1, dtype=dtype, device=DEV)
        kept = []
        for _ in range(2):  # factors as a product leaves them: act'(z) of z = x * 1, here of rows of one column
            x = rnd(g, m * n, 1, dtype=dtype)
            aux = torch.empty(lib.muon_hip_product_aux_bytes(_abi.dtype_code(dtype), m, n), dtype=torch.uint8, device=DEV)
            out = torch.empty_like(x)
            p = _abi.Product(kind=0, dtype=_abi.dtype_code(dtype), activation=3, m=m * n, n=1, k=1)
            p.a[:], p.a_row[:], p.a_col[:] = [x.data_ptr()] * 2, (1, 1), (1, 1)
            p.b[:], p.b_row[:], p.b_col[:] = [one.data_ptr()] * 2, (1, 1), (1, 1)
            p.out[0], p.aux[0] = out.data_ptr(), aux.data_ptr()
            need = lib.muon_hip_product_workspace(ctypes.addressof(p))
            ws = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
            _abi.check(lib.muon_hip_product_run(ctypes.addressof(p), ws.data_ptr(), need, _abi.stream_ptr(x.device)))
            kept.append((aux, R.activation("silu", x.double().view(m, n))[1]))
        pitch = n + 11
        for factors, results, sums in itertools.product((0, 1, 2), (True, False), (True, False)):
            dz = [torch.full((m, pitch), 7.0, dtype=dtype, device=DEV) for _ in range(max(1, factors))]
            db = [torch.full((n + 3,), 7.0, dtype=dtype, device=DEV) for _ in range(max(1, factors))]
            parts = torch.empty(lib.muon_hip_act_grad_partials(m, n) * max(1, factors), dtype=F, device=DEV)
            ptr = lambda ts, i, on: ts[i].data_ptr() if on and i < max(1, factors) else None
            _abi.check(lib.muon_hip_act_grad(dy.data_ptr(), factors, kept[0][0].data_ptr() if factors else None, kept[1][0].data_ptr() if factors > 1 else None,
                                             ptr(dz, 0, results), ptr(dz, 1, results), pitch, ptr(db, 0, sums), ptr(db, 1, sums), _abi.dtype_code(dtype),
                                             m, n, parts.data_ptr(), _abi.stream_ptr(dy.device)))
            for i in range(max(1, factors)):
                d = kept[i][1] if factors else torch.ones(m, n, dtype=torch.float64, device=DEV)
                want = dy.double() * d
                err = want.abs() * (R.cut(dtype) + 2 * R.F32) + dy.double().abs() * 2.0 ** -20 if factors else torch.zeros_like(want)
                if results:
                    R.check("dz", dz[i][:, :n], want, err + (R.unit(dtype) if factors else 0) * (want.abs() + err))
                assert (dz[i][:, n if results else 0:] == 7).all() and (db[i][n if sums else 0:] == 7).all()
                if sums:
                    total, room = want.sum(0), err.sum(0) + (m + 4) * R.F32 * (want.abs() + err).sum(0)
                    R.check("db", db[i][:n], total, room + R.unit(dtype) * (total.abs() + room))


def test_two_graphs_that_share_a_pool_and_replay_in_turn():
    g = gen_of(61)
    x, x2, w = rnd(g, 40, 4096), rnd(g, 40, 4096), rnd(g, 264, 4096, scale=0.02)
    E.linear(x, w, activation="silu")
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    pool = torch.cuda.graph_pool_handle()
    for gr, v in zip(graphs, (x, x2)):
        with torch.cuda.graph(gr, pool=pool):
            outs.append(E.linear(v, w, activation="silu"))
    for r in range(3):
        for v in (x, x2):
            v.copy_(rnd(g, 40, 4096))
        graphs[0].replay()
        graphs[1].replay()
        got = [o.clone() for o in outs]
        torch.cuda.synchronize()
        assert all(torch.equal(a, E.linear(v, w, activation="silu")) for a, v in zip(got, (x, x2))), r


def test_tensors_of_other_kinds_are_refused():
    class Mine(torch.Tensor):
        pass

    x, w = torch.zeros(4, 8, dtype=BF, device=DEV), torch.zeros(5, 8, dtype=BF, device=DEV)
    with pytest.raises(NotImplementedError, match="Mine"):
        E.linear(x.as_subclass(Mine), w)
    with pytest.raises(NotImplementedError, match="sparse"):
        E.linear(x.to_sparse(), w)
    with pytest.raises(TypeError, match="no tensor"):
        E.gated_linear(x, w, [1.0])
    with pytest.raises(TypeError, match="share one type"):
        E.linear(x, w.float())
    with pytest.raises(ValueError, match="do not fit"):
        E.linear(x, w[:, :7])


def test_values_behind_a_lazy_negation():
    """The imaginary part of a conjugate: the memory holds the values with the other sign."""
    z = torch.view_as_complex(torch.randn(6, 9, 2, device=DEV, generator=gen_of(47))).conj()
    assert z.imag.is_neg()
    w = torch.eye(9, device=DEV)
    assert torch.equal(E.linear(z.imag, w), z.imag.resolve_neg())
    assert torch.equal(E.linear(torch.zeros(6, 9, device=DEV), w, residual=z.imag), z.imag.resolve_neg())
    assert torch.equal(E.linear(w, z.imag), z.imag.resolve_neg().t())
