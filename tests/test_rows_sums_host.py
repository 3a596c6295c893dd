"""What the exact sums of rows_sums.py would let pass: no GPU needed."""
import pytest
import torch

from tests import rows_sums as S


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pattern", S.HOT)
def test_a_gradient_without_a_few_tokens_differs(pattern, dtype):
    tokens, vocab, n = 140000, 4000, 40
    g = torch.Generator().manual_seed(3)
    ids, dy = S.IDS[pattern](g, tokens, vocab), S.whole(g, tokens, n, dtype=dtype)
    want = S.embedding_grad(ids, dy, vocab, 0.5, S.padding(vocab)).to(dtype)
    hot = int(ids.mode().values)
    assert want[hot].any() and hot != S.padding(vocab)
    places = (ids == hot).nonzero().flatten()
    for left_out in (places[:137], places[-1:], places):  # as many as one chunk of sorted tokens, one, all
        some = dy.clone()
        some[left_out] = 0
        got = S.embedding_grad(ids, some, vocab, 0.5, S.padding(vocab)).to(dtype)
        # (one token of 140000 may be less than half a step of bf16)
        assert not torch.equal(got, want) or (dtype == torch.bfloat16 and len(left_out) == 1)
