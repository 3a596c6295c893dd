"""What the exact sums of rows_sums.py would let pass, and which kernels their cases run: no GPU needed."""
import pytest
import torch

from lmms_engine_amd import _abi
from tests import rows_sums as S
from tests.test_rows_host import kernel


def several(kind, dtype, rows, n):
    """Whether a workgroup has more than one turn, and the last one not for all of its rows at once; of streamed rows, more than one part."""
    r = _abi.norm_route(kind, dtype, rows, n, True)
    if r.pieces == 0:
        return r.groups > 1
    at_once = r.groups * (r.threads // r.lanes)
    return rows > at_once and rows % at_once != 0


def test_every_kernel_of_a_norms_gradient_takes_several_turns():
    sizes = [(m, n) for m in (70, 2000, 5000, 300000) for n in list(range(1, 200)) + list(range(200, 40000, 37)) + [2 ** i for i in range(17)]]
    for kind in (_abi.NORM_LAYER, _abi.NORM_RMS):
        for dtype in (_abi.F32, _abi.BF16):
            ran = {kernel(kind, dtype, m, n, True) for m, n in S.NORMS if several(kind, dtype, m, n)}
            there_are = {kernel(kind, dtype, m, n, True) for m, n in sizes}
            assert there_are <= ran, there_are - ran


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


@pytest.mark.parametrize("centred", [False, True])
def test_rows_of_ones_are_their_own_norms(centred):
    for n in (2, 250, 4096):
        x = S.rows_of_ones(torch.Generator().manual_seed(n), 50, n, centred, torch.float32)
        assert (x.abs() == 1).all() and (not centred or (x.sum(1) == 0).all())
        assert len(x.unique(dim=0)) > 1
