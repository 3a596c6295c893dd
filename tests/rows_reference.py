"""The formulas of the operators on rows in 64 bits, and how far the kernels may be from them.

A rounding to a type is off by at most u = eps / 2 of the value, one in fp32 by F = 2^-24.  A sum of n values over a row adds at most DEPTH(n) of them one
after the other (64 in a thread's registers, or n / 256 where a row is too long for them, and the threads of a row in a tree): it is off by at
most DEPTH(n) F of the sum of magnitudes.  A sum over m rows is off by at most m F of it."""
import numpy as np
import torch

F = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def DEPTH(n):
    return 96 + n / 256


def rounded(value, error, dtype):
    return value, error + unit(dtype) * (value.abs() + error)


def norm(kind, s, w, b, eps):
    """{name: (value, error before it is rounded)} of the norm of s and what its gradient reads."""
    n = s.size(-1)
    depth = (DEPTH(n) + 2) * F
    zero = torch.zeros_like(s[..., :1])
    if kind == "layer":
        mean, e_mean = s.mean(-1, keepdim=True), depth * s.abs().mean(-1, keepdim=True)
    else:
        mean, e_mean = zero, zero
    d = s - mean
    e_d = e_mean + F * (d.abs() + e_mean)
    square = (d * d).mean(-1, keepdim=True)
    e_square = depth * ((d.abs() + e_d) ** 2).mean(-1, keepdim=True) + (2 * d.abs() * e_d + e_d * e_d).mean(-1, keepdim=True)
    rstd = (square + eps) ** -0.5
    # (1 + t)^-1/2 is off from 1 by at most t for |t| <= 1/2; root, quotient, sum and eps itself are rounded
    t = e_square / (square + eps)
    assert bool((t <= 0.5).all() or not torch.isfinite(t).all()), "the input is no case for this bound"
    e_rstd = rstd * (t + 4 * F)
    hat = d * rstd
    e_hat = e_d * (rstd + e_rstd) + d.abs() * e_rstd + 2 * F * (hat.abs() + e_d * rstd)
    y, e_y = hat, e_hat
    if w is not None:
        y, e_y = hat * w, e_hat * w.abs() + F * (hat.abs() + e_hat) * w.abs()
    if b is not None:
        y = y + b
    e_y = e_y + 2 * F * (y.abs() + (b.abs() if b is not None else 0) + e_y)
    return {"y": (y, e_y), "hat": (hat, e_hat), "rstd": (rstd, e_rstd)}


def norm_grad(kind, s, w, eps, dy, ds):
    """{name: (value, error before it is rounded)} of the gradients."""
    n = s.size(-1)
    depth = (DEPTH(n) + 3) * F
    parts = norm(kind, s, None, None, eps)
    (hat, e_hat), (rstd, e_rstd) = parts["hat"], parts["rstd"]
    g = dy if w is None else dy * w
    c1, e_c1 = torch.zeros_like(rstd), torch.zeros_like(rstd)
    if kind == "layer":
        c1, e_c1 = g.mean(-1, keepdim=True), depth * g.abs().mean(-1, keepdim=True)
    c2 = (g * hat).mean(-1, keepdim=True)
    e_c2 = depth * (g.abs() * (hat.abs() + e_hat)).mean(-1, keepdim=True) + (g.abs() * e_hat).mean(-1, keepdim=True)
    inner = g - c1 - hat * c2
    e_inner = e_c1 + e_hat * (c2.abs() + e_c2) + hat.abs() * e_c2
    e_inner = e_inner + 5 * F * (g.abs() + c1.abs() + (hat * c2).abs() + e_inner)
    dx = rstd * inner
    e_dx = (rstd + e_rstd) * e_inner + inner.abs() * e_rstd + F * dx.abs()
    if ds is not None:
        dx = dx + ds
    e_dx = e_dx + 2 * F * (dx.abs() + e_dx)
    rows = s.numel() // max(1, n)
    over = tuple(range(s.dim() - 1))
    e_dw = (dy.abs() * e_hat + (rows + 4) * F * dy.abs() * (hat.abs() + e_hat)).sum(over)
    return {"dx": (dx, e_dx), "dw": ((dy * hat).sum(over), e_dw), "db": (dy.sum(over), (rows + 4) * F * dy.abs().sum(over))}


def embedding_grad(ids, dy, vocab, scale, skip=-1):
    device, ids, dy = dy.device, ids.cpu(), dy.cpu()  # (a GPU adds to one row in turn)
    dw, mag = (torch.zeros(vocab, dy.size(-1), dtype=torch.float64) for _ in range(2))
    count = torch.zeros(vocab, dtype=torch.float64)
    fine = (ids >= 0) & (ids < vocab) & (ids != skip)
    at = ids[fine].long()
    dw.index_add_(0, at, dy[fine] * scale)
    mag.index_add_(0, at, dy[fine].abs() * abs(scale))
    count.index_add_(0, at, torch.ones_like(at, dtype=torch.float64))
    return dw.to(device), ((count[:, None] + 3) * F * mag).to(device)


def philox(c, key):
    """Philox4x32-10 of numpy words; the published numbers are in test_rows_host.py."""
    c = [np.asarray(v, dtype=np.uint64) for v in c]
    low = np.uint64(0xFFFFFFFF)
    for r in range(10):
        k0, k1 = (key % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32, (key // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & low]
    return c


def numbers(count, seed, site, first=0):
    """The 32-bit number of each of `count` values from value `first`, a whole multiple of 8, on."""
    block = np.arange(first // 8, first // 8 + -(-count // 8), dtype=np.uint64)
    halves = []
    for which in (0, 1):
        words = philox([block & np.uint64(0xFFFFFFFF), block >> np.uint64(32), np.full_like(block, site), np.full_like(block, which)], seed % 2 ** 64)
        w = np.stack(words, axis=1)
        halves.append(np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], axis=2).reshape(-1)[:count])
    return (halves[0] << np.uint64(16)) | halves[1]


def dropout(x, p, seed, site, residual, dtype):
    """(value, error before it is rounded, kept) for x in 64 bits."""
    limit = int(np.rint(p * 2 ** 32))
    kept = torch.from_numpy(numbers(x.numel(), seed, site) >= limit).view(x.shape).to(x.device)
    scale = 2 ** 32 / (2 ** 32 - limit) if limit < 2 ** 32 else 0.0
    y = torch.where(kept, x * scale, torch.zeros_like(x))
    error = 2 * F * y.abs()
    if residual is not None:
        y = y + residual
        error = error + F * (y.abs() + error)
    return y, error, kept


def check(name, got, want, error, dtype=None):
    """Every value of `got` lies within `error` of the one wanted, rounded to dtype; where that is not finite, it is the same."""
    got = got.detach().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    if dtype is not None:
        want, error = rounded(want, error, dtype)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    assert torch.equal(got[~fine].nan_to_num(), want[~fine].nan_to_num()), name
    off = ((got - want).abs() - error)[fine]
    # (an error of zero is a value that is copied; 1e-37 stands for what underflows)
    assert not off.numel() or off.max().item() <= 1e-37, (name, off.max().item(), (got - want).abs()[fine].max().item())
