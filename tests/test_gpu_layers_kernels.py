"""Every kernel behind linear and gated_linear against the formulas in 64 bits: the cases of tests/layer_cases.py, x and the weights as rows and as
columns, with bias, activation and residual, every gradient."""
import itertools

import pytest
import torch

from lmms_engine_amd import _abi
from tests import layer_cases as cases
from tests import layer_reference as R
from tests.test_gpu_layers import compare, gen_of, rnd, run_gated, run_linear

pytestmark = pytest.mark.gpu
DTYPES = {_abi.BF16: torch.bfloat16, _abi.F32: torch.float32}


@pytest.mark.parametrize("layout", list(itertools.product((False, True), repeat=2)), ids=["rows-rows", "rows-columns", "columns-rows", "columns-columns"])
@pytest.mark.parametrize("case", cases.EVERY_KERNEL, ids=lambda c: "x".join(map(str, c[1:])) + ("-bf16" if c[0] == _abi.BF16 else "-f32"))
def test_every_kernel(case, layout):
    code, t, k, n = case
    dtype, g = DTYPES[code], gen_of(t + k + n)

    def matrix(rows, cols, scale, transposed):
        m = rnd(g, cols, rows, scale=scale, dtype=dtype).t() if transposed else rnd(g, rows, cols, scale=scale, dtype=dtype)
        return m.detach()

    x, w, w2 = matrix(t, k, 1.0, layout[0]), matrix(n, k, k ** -0.5, layout[1]), matrix(n, k, k ** -0.5, layout[1])
    b, b2, r, dy = rnd(g, n, dtype=dtype), rnd(g, n, dtype=dtype), rnd(g, t, n, dtype=dtype), rnd(g, t, n, dtype=dtype)
    name = ("gelu", "silu", "sigmoid", "gelu_tanh")[(t + k + n) % 4]
    compare(run_linear(x, w, b, r, name, dy), R.linear(x, w, b, r, name, dy, dtype))
    compare(run_gated(x.detach(), w.detach(), w2, b.detach(), b2, "silu", dy), R.gated(x, w, w2, b, b2, "silu", dy, dtype))
