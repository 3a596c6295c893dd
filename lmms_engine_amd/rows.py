"""What stands around the products of a model's blocks, row by row, forward and backward: its parameters are the other groups that `Muon` steps.

  embedding   rows of a table, times a scale
  layer_norm  (s - mean) / sqrt(var + eps) * weight + bias of s = x + residual
  rms_norm    s / sqrt(mean(s^2) + eps) * weight of s = x + residual
  dropout     residual + x / (1 - p) where a value is kept

A block of a transformer is then

    h, x = rms_norm(a, w_norm, residual=x)                             # the residual stream x takes up a, h is its norm
    h = gated_linear(h, w_gate, w_up)
    x = dropout(linear(h, w_down), 0.1, seed=step, site=layer, residual=x)

Tensors are float32 or bfloat16, one type per call (ids: 32-bit or 64-bit integers).  Everything is computed in float32 and rounded once; sums have
a fixed order, so the same call gives the same bits.  Rows are read as they lie where their values are back to back, other layouts through a
copy.  There is no counterpart in the reference, which leaves these to torch, and, as everywhere in this package, no CPU path.

The functions can be differentiated once by every floating tensor argument; what they keep is what the gradients of trained inputs read: a norm its
summed input, two floats a row and the weight, an embedding its ids, a dropout nothing (the mask is computed again).  Forward-mode differentiation,
second derivatives, tensor subclasses and recording (torch.jit.trace, make_fx, fake tensors) are refused; autocast leaves the calls alone.
"""
from __future__ import annotations

import operator
from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from . import _abi
from .layers import _check_one


def embedding(ids: Tensor, weight: Tensor, *, scale: float = 1.0, padding_idx: Optional[int] = None) -> Tensor:
    """weight[ids] * scale, of the shape [*ids.shape, n] for a weight of [vocab, n].

    An id outside of the table gives a row of NaN (the host would have to wait for the device to be told) and has no gradient.  The row
    `padding_idx` (from the end if negative) is looked up like any other and gets no gradient.  The weight's gradient is dense."""
    skip = -1
    if padding_idx is not None:
        vocab = weight.size(0) if isinstance(weight, Tensor) and weight.ndim else 0
        if not -vocab <= padding_idx < vocab:
            raise ValueError(f"padding_idx {padding_idx} is no row of a table of {vocab}")
        skip = padding_idx % vocab
    out = _abi.rows().embedding(ids, weight, scale, skip)
    if out is None:
        _check_one(weight, weight, "weight")
        _abi.dtype_code(weight.dtype)
        if weight.ndim != 2:
            raise ValueError(f"weight has shape {tuple(weight.shape)}, [vocab, n] is wanted")
        _check_whole(ids, weight, "ids", (torch.int32, torch.int64))
        _refuse(ids, weight)
    return out


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, *, eps: float = 1e-5,
               residual: Optional[Tensor] = None) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x [..., n]; weight and bias [n].

    With a residual, of the shape of x, the sum s = x + residual is normalised, as it is rounded to the tensors' type, and (y, s) is returned."""
    out = _abi.rows().norm(_abi.NORM_LAYER, x, weight, bias, residual, eps)
    if out is None:
        _refuse_norm(x, weight, bias, eps, residual)
    return out


def rms_norm(x: Tensor, weight: Optional[Tensor] = None, *, eps: float = 1e-6, residual: Optional[Tensor] = None) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension of x [..., n]; weight [n].  A residual is taken as in `layer_norm`."""
    out = _abi.rows().norm(_abi.NORM_RMS, x, weight, None, residual, eps)
    if out is None:
        _refuse_norm(x, weight, None, eps, residual)
    return out


def dropout(x: Tensor, p: float = 0.5, *, seed: Union[int, Tensor], site: int = 0, residual: Optional[Tensor] = None) -> Tensor:
    """residual + (x / (1 - p) where a value is kept, 0 where it is dropped), each value dropped with probability p.

    Which values are dropped depends on `seed`, `site` and a value's place in the row-major order of x's shape alone, so the backward pass draws the
    same again and no mask is kept.  Take another seed for every step and another site for every place in the model.  `seed` is a whole number of 64
    bits, or an int64 tensor of one element on x's device that is read when the kernels run (for a recorded HIP graph, whose replays would
    otherwise repeat one mask); it has to hold the same value in the backward pass.  `site` is a whole number below 2^32.  p is taken to 32 bits,
    and 1 / (1 - p) of what is taken."""
    if not isinstance(seed, Tensor):
        seed = operator.index(seed)
        if not -2 ** 63 <= seed < 2 ** 64:
            raise ValueError(f"seed {seed} is no number of 64 bits")
    if not 0 <= site < 2 ** 32:
        raise ValueError(f"site {site} is no number of 32 bits")
    out = _abi.rows().dropout(x, residual, p, seed, site)
    if out is None:
        if not 0 <= p <= 1:
            raise ValueError(f"p is {p}: a share from 0 to 1 is wanted")
        _check_like(x, residual)
        if isinstance(seed, Tensor):
            _check_whole(seed, x, "seed", (torch.int64,))
            if seed.numel() != 1:
                raise ValueError(f"seed has shape {tuple(seed.shape)}, one element is wanted")
        _refuse(x, residual, seed if isinstance(seed, Tensor) else None)
    return out


# ---- what the native calls leave to be refused ------------------------------------------------------


def _check_like(x: Tensor, residual: Optional[Tensor]) -> None:
    _check_one(x, x, "x")
    _abi.dtype_code(x.dtype)
    if residual is not None:
        _check_one(residual, x, "residual")
        if residual.shape != x.shape:
            raise ValueError(f"residual has shape {tuple(residual.shape)}, x {tuple(x.shape)}")


def _refuse_norm(x, weight, bias, eps, residual) -> None:
    if not eps >= 0:
        raise ValueError(f"eps is {eps}: a number that is not negative is wanted")
    _check_like(x, residual)
    if x.ndim < 1:
        raise ValueError("x needs at least one dimension")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _check_one(t, x, name)
            if t.shape != (x.size(-1),):
                raise ValueError(f"{name} has shape {tuple(t.shape)}, ({x.size(-1)},) is wanted")
    _refuse(x, weight, bias, residual)


def _check_whole(t: Tensor, like: Tensor, name: str, dtypes) -> None:
    _check_one(t, t, name)
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: {' or '.join(str(d) for d in dtypes)} is wanted, got {t.dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {like.device}")


def _refuse(*tensors) -> None:
    """Says why a call that fits by types and shapes was left alone."""
    for t in tensors:
        if t is not None and type(t) not in (Tensor, torch.nn.Parameter):
            raise NotImplementedError(f"plain tensors and parameters are taken, got {type(t).__name__}")
        if t is not None and t.layout != torch.strided:
            raise NotImplementedError(f"strided tensors are taken, got {t.layout}")
        if t is not None and t.numel() > 0 and t.untyped_storage().data_ptr() == 0:
            raise ValueError(f"the memory of a tensor of shape {tuple(t.shape)} was freed")
    raise ValueError(f"rows or columns are too many for one call: {[tuple(t.shape) for t in tensors if t is not None]}")
