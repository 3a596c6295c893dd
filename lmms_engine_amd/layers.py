"""The products of a model's layers, forward and backward, whose 2-D weights `Muon` trains.

  linear        act(x W^T + bias) + residual
  gated_linear  act(x Wg^T + bg) * (x Wu^T + bu), both projections in one kernel: the first half of a gated feed-forward block, whose
                second half is `linear` with the block's input as the residual

Each is one launch (two where a long reduction over few results is split) of the kernels behind muon_hip_product_run: matrix
instructions fed from LDS, sums, bias, activation and residual in fp32, one rounding.  Tensors are float32 or bfloat16, one type per call; the
products of float32 tensors keep single precision.  Operands are read as they lie, transposed views included; those whose rows are no whole
16-byte pieces go through packed copies.  There is no counterpart in the reference, which leaves its layers to torch, and, as everywhere in
this package, no CPU path.

Both functions can be differentiated once by every tensor argument.  For the backward pass they keep x where a weight is trained, the weights
where x has a gradient, and for every result the factors that the incoming gradient is multiplied by, of those that a trained input's
gradient reads: one with an activation, one for each projection of a gated pair, none otherwise, in 24 bits for bfloat16 tensors (three
bytes a value) and in 32 for float32.  Forward-mode differentiation, second derivatives, tensor subclasses and recording
(torch.jit.trace, make_fx, fake tensors) are refused; autocast leaves the calls alone, and modes that only watch torch operations
(counters, selective recomputation) see none of the products.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.distributed.tensor import DTensor

from . import _abi

ACTIVATIONS = tuple(_abi.ACTIVATIONS)


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *, activation: str = "none", residual: Optional[Tensor] = None) -> Tensor:
    """act(x @ weight.T + bias) + residual.

    x [..., k], weight [n, k], bias [n]; residual has the shape of the result, [..., n].  `activation` is one of ACTIVATIONS: none, relu,
    sigmoid, silu, gelu (with the error function) and gelu_tanh (torch's approximate="tanh")."""
    out = _abi.layers().linear(x, weight, bias, residual, _activation(activation))
    if out is None:
        n = _check(x, (weight,), (bias,))
        if residual is not None:
            _check_one(residual, x, "residual")
            if residual.shape != (*x.shape[:-1], n):
                raise ValueError(f"residual has shape {tuple(residual.shape)}, the result {(*x.shape[:-1], n)}")
        _refuse(x, weight, bias, residual)
    return out


def gated_linear(x: Tensor, weight_gate: Tensor, weight_up: Tensor, bias_gate: Optional[Tensor] = None, bias_up: Optional[Tensor] = None, *,
                 activation: str = "silu") -> Tensor:
    """act(x @ weight_gate.T + bias_gate) * (x @ weight_up.T + bias_up).

    x [..., k], weights [n, k], biases [n]; the result is [..., n].  `activation` as for `linear`."""
    out = _abi.layers().gated_linear(x, weight_gate, weight_up, bias_gate, bias_up, _activation(activation))
    if out is None:
        _check(x, (weight_gate, weight_up), (bias_gate, bias_up))
        _refuse(x, weight_gate, weight_up, bias_gate, bias_up)
    return out


# ---- what the native calls leave to be refused ------------------------------------------------------


def _activation(name: str) -> int:
    code = _abi.ACTIVATIONS.get(name)
    if code is None:
        raise ValueError(f"activation is one of {', '.join(ACTIVATIONS)}, got {name!r}")
    return code


def _check_one(t: Tensor, x: Tensor, name: str) -> None:
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} is no tensor: {type(t).__name__}")
    if not t.is_cuda:
        raise _abi.MuonHipError(f"{name} must live on a GPU: this build has no CPU path (got {t.device})")
    if isinstance(t, DTensor):
        raise NotImplementedError(f"{name} is a DTensor: one GPU, no collectives")
    if t.dtype != x.dtype:
        raise TypeError(f"x is {x.dtype}, {name} is {t.dtype}: the tensors of a layer share one type")
    if t.device != x.device:
        raise ValueError(f"x is on {x.device}, {name} on {t.device}")


def _check(x: Tensor, weights, biases) -> int:
    """Refuses what the kernels do not compute; the number of columns of the result."""
    _check_one(x, x, "x")
    _abi.dtype_code(x.dtype)
    if x.ndim < 1:
        raise ValueError("x needs at least one dimension")
    k = x.size(-1)
    n = weights[0].size(0) if weights[0].ndim else 0
    for w in weights:
        _check_one(w, x, "weight")
        if w.ndim != 2 or w.size(1) != k or w.size(0) != n:
            raise ValueError(f"weights {[tuple(v.shape) for v in weights]} do not fit x of shape {tuple(x.shape)}: [n, {k}] is wanted")
    for b in biases:
        if b is not None:
            _check_one(b, x, "bias")
            if b.shape != (n,):
                raise ValueError(f"bias has shape {tuple(b.shape)}, ({n},) is wanted")
    return n


def _refuse(*tensors) -> None:
    """Says why a call that fits by types and shapes was left alone."""
    for t in tensors:
        if t is not None and type(t) not in (Tensor, torch.nn.Parameter):
            raise NotImplementedError(f"linear and gated_linear take plain tensors and parameters, got {type(t).__name__}")
        if t is not None and t.layout != torch.strided:
            raise NotImplementedError(f"linear and gated_linear take strided tensors, got {t.layout}")
        if t is not None and t.numel() > 0 and t.untyped_storage().data_ptr() == 0:
            raise ValueError(f"the memory of a tensor of shape {tuple(t.shape)} was freed")
    raise ValueError(f"rows or columns are too many for one call: {[tuple(t.shape) for t in tensors if t is not None]}")
