"""Sums of the row operators' gradients that are exact whatever their order: of small whole numbers, which fp32 adds without rounding below 2^24.  A value that is
left out or counted twice, however many others there are, is one that differs."""
import torch

MOST = 8  # the largest magnitude of a value


def whole(g, *shape, dtype):
    return torch.randint(-MOST, MOST + 1, shape, generator=g, device=g.device).to(dtype)


def embedding_grad(ids, dy, vocab, scale, skip):
    """scale * the sum of dy over the tokens of each id, rounded once; scale is a power of two."""
    ids, dy = ids.cpu(), dy.cpu().double()
    assert MOST * ids.numel() < 2 ** 24
    fine = (ids >= 0) & (ids < vocab) & (ids != skip)
    return torch.zeros(vocab, dy.size(-1), dtype=torch.float64).index_add_(0, ids[fine].long(), dy[fine]) * scale


HOT = "one", "most of one", "two in turn"
IDS = {
    "any": lambda g, t, v: torch.randint(0, v, (t,), generator=g, device=g.device),
    "one": lambda g, t, v: torch.full((t,), v - 1, device=g.device),
    "most of one": lambda g, t, v: torch.where(torch.rand(t, generator=g, device=g.device) < 0.7, v // 2, torch.randint(0, v, (t,), generator=g, device=g.device)),
    "two in turn": lambda g, t, v: torch.arange(t, device=g.device) % 2 * (v - 1),
    "runs": lambda g, t, v: torch.arange(t, device=g.device) // 37 % v,
    "outside too": lambda g, t, v: torch.randint(-v, 2 * v, (t,), generator=g, device=g.device),
}
# (tokens, rows of the table, columns): one sorted list, several, more than are joined at once; rows of less than a piece
EMBEDDINGS = [(300, 17, 64), (5000, 50, 3), (8193, 11, 5), (9000, 20011, 96), (20001, 513, 264), (50000, 9, 7), (131073, 1000, 16), (140000, 4000, 40), (270001, 100, 1)]


def padding(vocab):
    """A row that has tokens, but none of the ids that HOT repeats."""
    return vocab // 3
