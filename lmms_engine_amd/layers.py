"""The products of a model's layers, forward and backward, whose 2-D weights `Muon` trains.

  linear        act(x W^T + bias) + residual
  gated_linear  act(x Wg^T + bg) * (x Wu^T + bu), both projections in one kernel: the first half of a gated feed-forward block, whose
                second half is `linear` with the block's input as the residual

Each is one launch (two where a long reduction over few results is split) of the kernels behind muon_hip_product_run: matrix
instructions fed from LDS, sums, bias, activation and residual in fp32, one rounding.  Tensors are float32 or bfloat16, one type per call; the
products of float32 tensors keep single precision.  Operands are read as they lie, transposed views included; those whose rows are no whole
16-byte pieces go through packed copies.  There is no counterpart in the reference, which leaves its layers to torch, and, as everywhere in
this package, no CPU path.

Both functions can be differentiated once by every tensor argument.  What the backward pass needs is kept in the tensors' type: the
inputs, and for every result the factors that the incoming gradient is multiplied by (nothing of the kind without an activation).
"""
from __future__ import annotations

import ctypes
from math import prod
from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable
from torch.distributed.tensor import DTensor

from . import _abi

ACTIVATIONS = tuple(_abi.ACTIVATIONS)


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *, activation: str = "none", residual: Optional[Tensor] = None) -> Tensor:
    """act(x @ weight.T + bias) + residual.

    x [..., k], weight [n, k], bias [n]; residual has the shape of the result, [..., n].  `activation` is one of ACTIVATIONS: none, relu,
    sigmoid, silu, gelu (with the error function) and gelu_tanh (torch's approximate="tanh")."""
    act = _activation(activation)
    n = _check(x, (weight,), (bias,))
    shape = (*x.shape[:-1], n)
    if residual is not None:
        _check_one(residual, x, "residual")
        if residual.shape != shape:
            raise ValueError(f"residual has shape {tuple(residual.shape)}, the result {shape}")
    if torch.is_grad_enabled() and _any_grad(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, act)
    return _linear(x, weight, bias, residual, act, shape, False)[0]


def gated_linear(x: Tensor, weight_gate: Tensor, weight_up: Tensor, bias_gate: Optional[Tensor] = None, bias_up: Optional[Tensor] = None, *,
                 activation: str = "silu") -> Tensor:
    """act(x @ weight_gate.T + bias_gate) * (x @ weight_up.T + bias_up).

    x [..., k], weights [n, k], biases [n]; the result is [..., n].  `activation` as for `linear`."""
    act = _activation(activation)
    n = _check(x, (weight_gate, weight_up), (bias_gate, bias_up))
    if torch.is_grad_enabled() and _any_grad(x, weight_gate, weight_up, bias_gate, bias_up):
        return _GatedLinear.apply(x, weight_gate, weight_up, bias_gate, bias_up, act)
    return _gated(x, weight_gate, weight_up, bias_gate, bias_up, act, (*x.shape[:-1], n), False)[0]


# ---- arguments -------------------------------------------------------------------------------


def _activation(name: str) -> int:
    code = _abi.ACTIVATIONS.get(name)
    if code is None:
        raise ValueError(f"activation is one of {', '.join(ACTIVATIONS)}, got {name!r}")
    return code


def _any_grad(*tensors) -> bool:
    return any(t is not None and t.requires_grad for t in tensors)


def _check_one(t: Tensor, x: Tensor, name: str) -> None:
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


def _rows(t: Tensor) -> Tensor:
    """t as a matrix of its last dimension's rows: a view where there is one.  Its values are where its pointer says."""
    return t.detach().resolve_neg().reshape(prod(t.shape[:-1]), t.size(-1))


def _dense(t: Optional[Tensor]) -> Optional[Tensor]:
    return None if t is None else t.detach().resolve_neg().contiguous()


class _On:
    """The tensor's device as the current one, while it is not already."""

    def __init__(self, t: Tensor):
        self.device = None if t.get_device() == torch.cuda.current_device() else torch.cuda.device(t.device)

    def __enter__(self):
        if self.device is not None:
            self.device.__enter__()

    def __exit__(self, *exc):
        if self.device is not None:
            self.device.__exit__(*exc)


# ---- launches ---------------------------------------------------------------------------------


def _ptr(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


def _operands(*matrices, turned: bool = False):
    """Pointers, strides of the row index and strides of the reduction index of one or two matrices; turned: the reduction runs down
    the columns."""
    r, c = (1, 0) if turned else (0, 1)
    more = matrices[1:] or matrices
    pair = (matrices[0], more[0])
    return ([t.data_ptr() for t in pair], [t.stride(r) for t in pair], [t.stride(c) for t in pair])


def _run(kind: int, like: Tensor, m: int, n: int, k: int, a, b, out, act: int = 0, bias=(None, None), residual: Optional[Tensor] = None,
         aux=(None, None)) -> None:
    """One product on the current device and stream."""
    lib = _abi.lib()
    p = _abi.Product(kind=kind, dtype=_abi.dtype_code(like.dtype), activation=act, m=m, n=n, k=k)
    p.a[:], p.a_row[:], p.a_col[:] = a
    p.b[:], p.b_row[:], p.b_col[:] = b
    p.out[:] = (out[0].data_ptr(), _ptr(out[1]) if len(out) > 1 else None)
    if bias[0] is not None or bias[1] is not None:
        p.bias[:] = (_ptr(bias[0]), _ptr(bias[1]))
    if residual is not None:
        p.residual, p.res_row, p.res_col = residual.data_ptr(), residual.stride(0), residual.stride(1)
    if aux[0] is not None:
        p.aux[:] = (_ptr(aux[0]), _ptr(aux[1]))
    at = ctypes.addressof(p)
    need = lib.muon_hip_product_workspace(at)
    if need < 0:
        _abi.check(need, "product")
    ws = torch.empty(need, dtype=torch.uint8, device=like.device) if need else None
    _abi.check(lib.muon_hip_product_run(at, _ptr(ws), need, _abi.stream_ptr(like.device)), "product")


def _linear(x, weight, bias, residual, act, shape, keep):
    """The result, and act'(.) where it is to be kept."""
    x2, w = _rows(x), weight.detach().resolve_neg()
    m, k = x2.shape
    n = w.size(0)
    r = None if residual is None else _rows(residual)
    with _On(x):
        out = torch.empty(shape, dtype=x.dtype, device=x.device)
        d = torch.empty((m, n), dtype=x.dtype, device=x.device) if keep and act else None
        _run(_abi.PRODUCT_LINEAR, x, m, n, k, _operands(x2), _operands(w), (out,), act, (_dense(bias), None), r, (d, None))
    return out, d


def _gated(x, weight_gate, weight_up, bias_gate, bias_up, act, shape, keep):
    """The result, and act(g) and u act'(g) where they are to be kept."""
    x2, wg, wu = _rows(x), weight_gate.detach().resolve_neg(), weight_up.detach().resolve_neg()
    m, k = x2.shape
    n = wg.size(0)
    with _On(x):
        out = torch.empty(shape, dtype=x.dtype, device=x.device)
        s, t = (torch.empty((m, n), dtype=x.dtype, device=x.device) for _ in range(2)) if keep else (None, None)
        _run(_abi.PRODUCT_GATED, x, m, n, k, _operands(x2), _operands(wg, wu), (out,), act, (_dense(bias_gate), _dense(bias_up)), None, (s, t))
    return out, s, t


def _act_grad(dy: Tensor, d0: Optional[Tensor], d1: Optional[Tensor], want_dz: bool, want_db):
    """dz = dy * d for one or two factors (dy itself where there is none and its rows are whole 16-byte pieces) and their sums over the
    rows where those are wanted, on the current device."""
    m, n = dy.shape
    pitch = -(-n // 8) * 8
    pair = d1 is not None
    make = want_dz and (d0 is not None or pitch != n or dy.data_ptr() % 16 != 0)
    dz = [torch.empty((m, pitch), dtype=dy.dtype, device=dy.device)[:, :n] for _ in range(1 + pair)] if make else [dy] * (1 + pair)
    db = [torch.empty(n, dtype=dy.dtype, device=dy.device) if w else None for w in want_db]
    if make or any(want_db):
        lib = _abi.lib()
        floats = lib.muon_hip_act_grad_partials(m, n) * (1 + pair) if any(want_db) else 0
        parts = torch.empty(floats, dtype=torch.float32, device=dy.device) if floats else None
        z = [_ptr(t) for t in dz] if make else [None]
        _abi.check(lib.muon_hip_act_grad(dy.data_ptr(), (d0 is not None) + pair, _ptr(d0), _ptr(d1), z[0], z[1] if pair and make else None, pitch, _ptr(db[0]),
                                         _ptr(db[1]) if pair else None, _abi.dtype_code(dy.dtype), m, n, _ptr(parts),
                                         _abi.stream_ptr(dy.device)), "act_grad")
    return dz, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        keep = any(ctx.needs_input_grad[:3])
        out, d = _linear(x, weight, bias, residual, act, (*x.shape[:-1], weight.size(0)), keep)
        ctx.save_for_backward(x, weight, d)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, d = ctx.saved_tensors
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if want_x or want_w or want_b:
            x2, w = _rows(x), weight.detach().resolve_neg()
            (m, k), n = x2.shape, w.size(0)
            with _On(x):
                (dz,), (db,) = _act_grad(_dense(dy).view(m, n), d, None, want_x or want_w, (want_b,))
                if want_x:
                    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
                    _run(_abi.PRODUCT_LINEAR, x, m, k, n, _operands(dz), _operands(w, turned=True), (dx,))
                if want_w:
                    dw = torch.empty((n, k), dtype=x.dtype, device=x.device)
                    _run(_abi.PRODUCT_LINEAR, x, n, k, m, _operands(dz, turned=True), _operands(x2, turned=True), (dw,))
        return dx, dw, db, dy if want_r else None, None


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight_gate, weight_up, bias_gate, bias_up, act):
        out, s, t = _gated(x, weight_gate, weight_up, bias_gate, bias_up, act, (*x.shape[:-1], weight_gate.size(0)), True)
        ctx.save_for_backward(x, weight_gate, weight_up, s, t)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, weight_gate, weight_up, s, t = ctx.saved_tensors
        want_x, want_wg, want_wu, want_bg, want_bu = ctx.needs_input_grad[:5]
        x2, wg, wu = _rows(x), weight_gate.detach().resolve_neg(), weight_up.detach().resolve_neg()
        (m, k), n = x2.shape, wg.size(0)
        dx, dwg, dwu = None, None, None
        with _On(x):
            (dg, du), (dbg, dbu) = _act_grad(_dense(dh).view(m, n), t, s, want_x or want_wg or want_wu, (want_bg, want_bu))
            if want_x:
                dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
                _run(_abi.PRODUCT_SUM, x, m, k, n, _operands(dg, du), _operands(wg, wu, turned=True), (dx,))
            if want_wg and want_wu:
                dwg, dwu = (torch.empty((n, k), dtype=x.dtype, device=x.device) for _ in range(2))
                _run(_abi.PRODUCT_EACH, x, n, k, m, _operands(dg, du, turned=True), _operands(x2, turned=True), (dwg, dwu))
            elif want_wg or want_wu:
                dw = torch.empty((n, k), dtype=x.dtype, device=x.device)
                _run(_abi.PRODUCT_LINEAR, x, n, k, m, _operands(dg if want_wg else du, turned=True), _operands(x2, turned=True), (dw,))
                dwg, dwu = (dw, None) if want_wg else (None, dw)
        return dx, dwg, dwu, dbg, dbu, None
