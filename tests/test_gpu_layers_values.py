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
