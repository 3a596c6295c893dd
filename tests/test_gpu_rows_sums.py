"""Sums over rows and over tokens, exact (rows_sums.py): norms' weights over many rows, tables' gradients over ids that have many tokens."""
import pytest
import torch

import lmms_engine_amd as E
from tests import rows_sums as S
from tests.test_gpu_rows import DEV, DTYPES, compare_norm, gen_of, rnd, run_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,n", S.NORMS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_gradients_of_norms_over_many_rows(kind, dtype, rows, n):
    g = gen_of(kind, dtype, rows, n)
    x = S.rows_of_ones(g, rows, n, kind == "layer", dtype)
    w, b = S.whole(g, n, dtype=dtype), torch.zeros(n, dtype=dtype, device=DEV) if kind == "layer" else None
    dy, ds = S.whole(g, rows, n, dtype=dtype), rnd(g, rows, n, dtype=dtype)
    assert S.MOST * rows < 2 ** 24 and n < 2 ** 24
    for residual in (None, torch.zeros_like(x)):
        got = run_norm(kind, x, w, b, residual, 0.0, dy, ds)
        assert torch.equal(got["dw"], (dy.double() * x.double()).sum(0).to(dtype))
        if b is not None:
            assert torch.equal(got["db"], dy.double().sum(0).to(dtype))
        compare_norm(kind, x, w, b, residual, 0.0, dy, ds, {k: v for k, v in got.items() if k in ("y", "s", "dx", "dr")})


@pytest.mark.parametrize("pattern", list(S.IDS))
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,vocab,n", S.EMBEDDINGS)
def test_gradients_of_embeddings_of_many_tokens(tokens, vocab, n, dtype, pattern):
    g = gen_of(tokens, vocab, n, dtype, pattern)
    ids, dy = S.IDS[pattern](g, tokens, vocab), S.whole(g, tokens, n, dtype=dtype)
    for scale, skip in ((1.0, None), (0.5, S.padding(vocab))):
        w = rnd(g, vocab, n, dtype=dtype).requires_grad_(True)
        (dw,) = torch.autograd.grad(E.embedding(ids, w, scale=scale, padding_idx=skip), w, dy)
        assert torch.equal(dw.cpu(), S.embedding_grad(ids, dy, vocab, scale, -1 if skip is None else skip).to(dtype))
