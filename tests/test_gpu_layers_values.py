"""Values of activations and of what is kept for the backward pass, relative to themselves."""
import ctypes

import pytest
import torch

import lmms_engine_amd as E
from lmms_engine_amd import _abi
from tests import layer_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F], ids=["bf16", "f32"])
def test_the_lower_tail_of_gelu_is_right_to_its_own_size(dtype):
    """z Phi(z) and its derivative from -2 down to where they leave the normal numbers, where both are far smaller than an absolute bound tells.

    In fp32 the argument of the exponential, at most 126 in powers of two, is off by two roundings (126 * 2^-23 * ln 2 < 2^-16 of the value);
    for fp32 tensors z^2 / 2 is rounded too and erfc carries a rounding of its argument on with a slope of z^2 <= 170 (2^-16 again).  Phi itself
    may be off by another 2^-15, the derivative, a difference of two parts of which the larger is at most 1.6 times itself, by twice as much.
    The result is rounded; so are dz, of a factor cut off behind 16 bits of its significand (bf16 tensors), and dx, which is dz itself."""
    z = torch.linspace(-12.5, -2, 2000).to(dtype).unique().to(DEV)[:, None].requires_grad_(True)
    one = torch.ones(1, 1, dtype=dtype, device=DEV)
    y = E.linear(z, one, activation="gelu")
    (dz,) = torch.autograd.grad(y, z, torch.ones_like(y))
    a, d = R.activation("gelu", z.detach().double())
    u = R.unit(dtype)
    for name, got, want, room in (("y", y, a, u + 2.0 ** -14), ("dz", dz, d, u + R.cut(dtype) + 2.0 ** -13)):
        off = ((got.detach().double() - want).abs() / want.abs()).max().item()
        assert off <= room, (name, off, room)
    h = E.gated_linear(z.detach(), one, one, activation="gelu")
    off = ((h.double() - a * z.detach().double()).abs() / (a * z.detach().double()).abs()).max().item()
    assert off <= u + 2.0 ** -14, off


def test_factors_are_rounded_to_the_bits_that_are_kept():
    """24 bits of a factor, 16 of them its significand's: off by half a step of theirs, 2^-16 of the value, to either side.  Two rows' factors differ
    by less than a bf16 value shows, and their difference is what is left of the bias's gradient."""
    tiny = 2.0 ** -15
    for part in (255 / 256, 129 / 256, 127 / 256, 3 / 256):
        x = torch.tensor([[1.0, part * tiny], [1.0, 0.0]], dtype=BF, device=DEV)
        w = torch.ones(8, 2, dtype=BF, device=DEV)
        bg = torch.zeros(8, dtype=BF, device=DEV, requires_grad=True)
        h = E.gated_linear(x, w, w, bg, None, activation="none")  # the factor of bg's gradient is x w^T: 1 + part * 2^-15 and 1, exact sums
        (db,) = torch.autograd.grad(h, bg, torch.tensor([[1.0], [-1.0]], dtype=BF, device=DEV).expand(2, 8))
        off = (db.double() - part * tiny).abs().max().item()
        assert off <= 2.0 ** -16 * (1 + tiny) + 2.0 ** -9 * tiny, (part, off)


@pytest.mark.parametrize("dtype", [BF, F], ids=["bf16", "f32"])
@pytest.mark.parametrize("size", [(3, 40, 24), (70, 64, 75), (300, 2000, 40)], ids=str)
def test_a_product_without_an_activation_keeps_its_factor_too(size, dtype):
    """act'(.) is 1 where there is none: whoever asks for it gets it."""
    t, k, n = size
    g = torch.Generator(device=DEV).manual_seed(2)
    lib, code = _abi.lib(), _abi.dtype_code(dtype)
    x, w, dy = (torch.randn(*s, generator=g, device=DEV).to(dtype) for s in ((t, k), (n, k), (t, n)))
    out, dz = torch.empty(t, n, dtype=dtype, device=DEV), torch.empty(t, n, dtype=dtype, device=DEV)
    aux = torch.zeros(lib.muon_hip_product_aux_bytes(code, t, n), dtype=torch.uint8, device=DEV)
    p = _abi.Product(kind=_abi.PRODUCT_LINEAR, dtype=code, m=t, n=n, k=k)
    p.a[0], p.a_row[0], p.a_col[0] = x.data_ptr(), k, 1
    p.b[0], p.b_row[0], p.b_col[0] = w.data_ptr(), k, 1
    p.out[0], p.aux[0] = out.data_ptr(), aux.data_ptr()
    need = lib.muon_hip_product_workspace(ctypes.addressof(p))
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
    stream = _abi.stream_ptr(x.device)
    _abi.check(lib.muon_hip_product_run(ctypes.addressof(p), ws.data_ptr(), need, stream))
    _abi.check(lib.muon_hip_act_grad(dy.data_ptr(), 1, aux.data_ptr(), None, dz.data_ptr(), None, n, None, None, code, t, n, None, stream))
    assert torch.equal(dz, dy) and torch.equal(out, E.linear(x, w))


def test_launches_at_the_limit_of_a_grid():
    """Few rows against 2^27 rows of a table, for which the walk over it has more threads than a launch; sums over 2^30 rows, for which 64 rows to a
    workgroup would be."""
    n, k = 2 ** 27 + 24, 8
    g = torch.Generator(device=DEV).manual_seed(4)
    x, w = (torch.randint(-4, 5, s, generator=g, device=DEV, dtype=torch.int8).to(BF) for s in ((3, k), (n, k)))
    y, h = E.linear(x, w), E.gated_linear(x, w, w, activation="none")
    for at in (slice(0, 100), slice(2 ** 26, 2 ** 26 + 100), slice(n - 100, n)):
        want = x.double() @ w[at].double().t()  # whole numbers below 2^8, and their squares, rounded once
        assert torch.equal(y[:, at].double(), want) and torch.equal(h[:, at], want.square().to(BF))
    del w, y, h
    m = 2 ** 30 + 9
    part = torch.randint(-1, 2, (2 ** 20, 1), generator=g, device=DEV, dtype=torch.int8).float()
    dy = torch.cat([part.repeat(2 ** 10, 1), part[:9]])
    b = torch.zeros(1, device=DEV, requires_grad=True)
    (db,) = torch.autograd.grad(E.linear(torch.zeros(m, 1, device=DEV), torch.zeros(1, 1, device=DEV), b), b, dy)
    assert db.item() == part.sum().item() * 2 ** 10 + part[:9].sum().item()  # (every partial sum is a whole number below 2^24)
