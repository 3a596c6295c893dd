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


def rows_of_ones(g, rows, n, centred, dtype):
    """Values of 1 and -1, of a centred row as many of either: mean 0, mean of squares 1, so that with eps = 0 a norm's hat is its input, exactly."""
    if not centred:
        return torch.where(torch.rand(rows, n, generator=g, device=g.device) < 0.5, 1.0, -1.0).to(dtype)
    assert n % 2 == 0
    first = torch.where(torch.rand(rows, n // 2, generator=g, device=g.device) < 0.5, 1.0, -1.0)
    x = torch.cat([first, -first], 1)
    return x[:, torch.randperm(n, generator=g, device=g.device)].to(dtype)


# (rows, columns), columns even: test_rows_sums_host.py holds the list to giving a workgroup of every kernel of a norm's gradient several turns, or several parts
# to a sum over columns, with a rest behind them
NORMS = [(150001, 2), (90001, 6), (40003, 30), (40003, 128), (20003, 250), (20003, 256), (12003, 506), (12003, 512), (7003, 1002), (7003, 1024), (3001, 4096), (3001, 4098),
         (2001, 8192), (2001, 8194), (1501, 12288), (1501, 12290), (1301, 16382), (1301, 16384), (300, 20000), (203, 33002)]

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
