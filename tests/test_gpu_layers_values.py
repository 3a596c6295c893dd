"""Values of activations and of what is kept for the backward pass, relative to themselves."""
import ctypes
import itertools

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
