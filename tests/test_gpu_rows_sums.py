"""Sums over tokens, exact (rows_sums.py): tables' gradients over ids that have many tokens."""
import pytest
import torch

import lmms_engine_amd as E
from tests import rows_sums as S
from tests.test_gpu_rows import DTYPES, gen_of, rnd

pytestmark = pytest.mark.gpu


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
