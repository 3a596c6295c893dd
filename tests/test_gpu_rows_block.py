"""A small language model of embedding, dropout, norms, linear and gated_linear, forward and backward, and the optimizer on its parameters."""
import numpy as np
import pytest
import torch

import lmms_engine_amd as E
from lmms_engine_amd.clip_grad import clip_grad_norm_
from tests import rows_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
VOCAB, WIDTH, INNER, TOKENS, LAYERS, P, SEED = 203, 136, 264, 150, 2, 0.15, 42
PLACEHOLDER = 199


def parameters(dtype):
    g = torch.Generator(device=DEV).manual_seed(5)

    def make(*shape, scale=1.0, at=0.0):
        return torch.nn.Parameter((torch.randn(*shape, generator=g, device=DEV) * scale + at).to(dtype))

    p = {"table": make(VOCAB, WIDTH, scale=0.5), "out_norm": make(WIDTH, scale=0.1, at=1.0), "out_bias": make(WIDTH, scale=0.1)}
    for i in range(LAYERS):
        p.update({f"norm{i}": make(WIDTH, scale=0.1, at=1.0), f"gate{i}": make(INNER, WIDTH, scale=WIDTH ** -0.5), f"up{i}": make(INNER, WIDTH, scale=WIDTH ** -0.5),
                  f"down{i}": make(WIDTH, INNER, scale=INNER ** -0.5)})
    return p


def tokens():
    g = torch.Generator(device=DEV).manual_seed(6)
    ids = torch.randint(0, 150, (TOKENS,), generator=g, device=DEV)
    ids[20:90] = PLACEHOLDER
    return ids.view(2, TOKENS // 2)


def model(p, ids, seed):
    """Hidden states of the last layer's norm."""
    x = E.dropout(E.embedding(ids, p["table"], scale=WIDTH ** 0.5), P, seed=seed, site=0)
    h = E.rms_norm(x, p["norm0"])
    for i in range(LAYERS):
        a = E.linear(E.gated_linear(h, p[f"gate{i}"], p[f"up{i}"]), p[f"down{i}"])
        a = E.dropout(a, P, seed=seed, site=i + 1)
        if i + 1 < LAYERS:
            h, x = E.rms_norm(a, p[f"norm{i + 1}"], residual=x)
        else:
            h, x = E.layer_norm(a, p["out_norm"], p["out_bias"], residual=x)
    return E.linear(h, p["table"])  # the head shares the embedding's table


def wide_model(p, ids, seed):
    def dropped(x, site):
        limit = int(np.rint(P * 2 ** 32))
        kept = torch.from_numpy(R.numbers(x.numel(), seed, site) >= limit).view(x.shape).to(DEV)
        return x * kept * (2 ** 32 / (2 ** 32 - limit))

    def rms(x, w):
        return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w

    x = dropped(p["table"][ids] * WIDTH ** 0.5, 0)
    h = rms(x, p["norm0"])
    for i in range(LAYERS):
        g = h @ p[f"gate{i}"].t()
        x = x + dropped((g * torch.sigmoid(g) * (h @ p[f"up{i}"].t())) @ p[f"down{i}"].t(), i + 1)
        if i + 1 < LAYERS:
            h = rms(x, p[f"norm{i + 1}"])
    h = (x - x.mean(-1, keepdim=True)) * (x.var(-1, unbiased=False, keepdim=True) + 1e-5).rsqrt() * p["out_norm"] + p["out_bias"]
    return h @ p["table"].t()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_model_and_its_gradients(dtype):
    """Every stage rounds its result once, by half a step of it at most; there are 14 on the longest way forward and as many back.  In fp32 a stage's
    sums, of up to 264 values, weigh more: 268 roundings of 2^-24 at most."""
    p, ids = parameters(dtype), tokens()
    wide = {k: v.detach().double().requires_grad_(True) for k, v in p.items()}
    y, want = model(p, ids, SEED), wide_model(wide, ids, SEED)
    g = torch.Generator(device=DEV).manual_seed(7)
    dy = torch.randn(y.shape, generator=g, device=DEV).to(dtype)
    grads = torch.autograd.grad(y, list(p.values()), dy)
    expected = torch.autograd.grad(want, list(wide.values()), dy.double())
    stage = R.unit(dtype) + (268 * R.F if dtype == torch.float32 else 0)
    assert (y.double() - want).norm() <= 14 * stage * want.norm()
    for name, a, e in zip(p, grads, expected):
        assert a.shape == e.shape and (a.double() - e).norm() <= 28 * stage * e.norm(), (name, ((a.double() - e).norm() / e.norm()).item())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_optimizer_steps_what_the_model_is_made_of(dtype):
    p, ids = parameters(dtype), tokens()
    before = {k: v.detach().clone() for k, v in p.items()}
    matrices = [v for k, v in p.items() if v.ndim == 2 and k != "table"]
    others = [v for k, v in p.items() if v.ndim < 2 or k == "table"]
    opt = E.Muon([dict(params=matrices, use_muon=True, lr=0.02, momentum=0.95, weight_decay=0.0, rms_scale=False),
                  dict(params=others, use_muon=False, lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.0)])
    # lookups alone, so that rows of the table without tokens have no gradient
    for step in range(2):
        opt.zero_grad()
        x = E.dropout(E.embedding(ids, p["table"], padding_idx=PLACEHOLDER), P, seed=step, site=0)
        h, x = E.layer_norm(x, p["norm0"], p["out_bias"], residual=x)
        a = E.linear(E.gated_linear(h, p["gate0"], p["up0"]), p["down0"])
        h, x = E.rms_norm(E.dropout(a, P, seed=step, site=1), p["out_norm"], residual=x)
        h.float().square().mean().add(x.float().square().mean()).backward()
        total = clip_grad_norm_([v for v in p.values() if v.grad is not None], 1.0)
        assert torch.isfinite(total) and total > 0
        opt.step()
    seen = torch.zeros(VOCAB, dtype=torch.bool, device=DEV)
    seen[ids.flatten()] = True
    seen[PLACEHOLDER] = False
    changed = (p["table"] != before["table"]).any(1)
    assert torch.equal(changed, seen)
    for name in ("norm0", "out_norm", "out_bias", "gate0", "up0", "down0"):
        assert torch.isfinite(p[name]).all() and bool((p[name] != before[name]).any()), name
