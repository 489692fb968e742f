"""Prompts of random sizes, gates, keys and values, up to 2^60 apart, against a 64-bit token loop.

Tolerances: the state as in test_gated_delta_gpu.py, row by row; o within the same share (24 sqrt(T) 2^-24) of scale |q| times the
largest norm that the state's row has or, but for its decays, had, plus half a step of its type.  Sizes below 1e-28 are left out:
there fp32's smallest numbers are what counts."""
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

D = torch.float64


def loop(x, lens, scale, norm):
    """o, states, and the norms of the states' rows, each the largest that its decays since have left, at every token and at the end."""
    q, k, v, a, b = (x[n].to(D) for n in "qkvab")
    if norm:
        q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-6) for t in (q, k))
    rep = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    keep = torch.exp(-torch.exp(x["A_log"].to(D)) * torch.nn.functional.softplus(a + x["dt_bias"].to(D), threshold=40))
    beta, S = torch.sigmoid(b), x["state"].to(D).clone()
    first = np.concatenate([[0], np.cumsum(lens)])
    o, size, held = torch.zeros_like(v), torch.zeros_like(v), S.norm(dim=-1)
    for t in range(max(lens)):
        i = torch.tensor([j for j, n in enumerate(lens) if n > t], device="cuda")
        r = torch.tensor([first[j] + t for j, n in enumerate(lens) if n > t], device="cuda")
        old = keep[r][:, :, None, None] * S[i]
        u = beta[r][:, :, None] * (v[r] - (old * k[r][:, :, None, :]).sum(-1))
        S[i] = old + u[..., None] * k[r][:, :, None, :]
        o[r] = scale * (S[i] * q[r][:, :, None, :]).sum(-1)
        rows = torch.maximum(torch.maximum(S[i].norm(dim=-1), old.norm(dim=-1)), u.abs() * k[r].norm(dim=-1)[..., None])
        held[i] = torch.maximum(keep[r][:, :, None] * held[i], rows)
        size[r] = scale * held[i] * q[r].norm(dim=-1)[..., None]
    return o, S, size, held


def draw(seed, dtype):
    rng, g = random.Random(seed), torch.Generator("cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    hk, hv, dk, dv = rng.choice([(1, 2, 128, 32), (2, 4, 64, 48), (2, 40, 128, 64), (1, 4, 128, 128), (2, 2, 64, 256)])
    lens = [rng.choice([13, 20, 33, 64, 65, 100, 128, 150]) for _ in range(rng.choice([1, 2, 4]))]
    n, norm, silu = sum(lens), rng.random() < 0.75, torch.nn.functional.silu
    q, k, v = silu(randn(n, hk, dk)), silu(randn(n, hk, dk)), silu(randn(n, hv, dv))
    span = rng.choice([0, 0.3, 0.6, 1]) * (20 if dtype is torch.float16 else rng.choice([20, 40, 60]))
    shape = rng.choice([(n, 1, 1), (1, hv, dv), (n, hv, dv), None])
    v *= 2.0 ** (-span * (rand(*shape) if shape else rand((n + 7) // 8, 1, 1).repeat_interleave(8, 0)[:n]))
    if rng.random() < 0.3:
        v *= rand(n, hv, 1) < 0.5
    if norm:
        k, q = k * 2.0 ** (rng.choice([0, 3, 8, 16]) * (rand(n, hk, 1) - 0.5)), q * 2.0 ** (rng.choice([0, 8]) * (rand(n, hk, 1) - 0.5))
        if rng.random() < 0.3:
            k *= rand(n, hk, 1) < 0.9
    else:
        k = k / k.norm(dim=-1, keepdim=True) * 2.0 ** (-rng.choice([0, 4, 10]) * rand(n, hk, 1))
        q = q / q.norm(dim=-1, keepdim=True)
    a = rng.choice([0, -8, -3, 2]) + rng.choice([0, 1, 4]) * randn(n, hv)
    b = rng.choice([0, -6, 3]) + rng.choice([1, 4]) * randn(n, hv)
    if rng.random() < 0.5:
        a = torch.where(rand(n, hv) < rng.choice([0.02, 0.1]), 60.0, a)
    if rng.random() < 0.3:
        b = torch.where(rand(n, hv) < 0.1, -30.0, b)
    v *= rng.choice([1, 1e3, 3e4]) if dtype is torch.float16 else rng.choice([1, 1e6, 1e-6])
    most = torch.finfo(dtype).max
    x = {m: t.clamp(-most, most).to(dtype) for m, t in (("q", q), ("k", k), ("v", v), ("a", a), ("b", b))}
    x["A_log"], x["dt_bias"] = torch.log(0.1 + 15 * rand(hv)), -6 + 4 * rand(hv)
    x["state"] = randn(len(lens), hv, dv, dk) * rng.choice([0, 0.3, 1e-4, 1e3, 1e6])
    return x, lens, norm


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("seed", range(60))
def test_random_prompts(seed, dtype):
    from dfssm_b200 import ops
    x, lens, norm = draw(1000 * (dtype is torch.float16) + seed, dtype)
    want, S, size, held = loop(x, lens, 0.1, norm)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    o = ops.gated_delta_prefill(*(x[n] for n in ("q", "k", "v", "a", "b", "A_log", "dt_bias", "state")), cu, scale=0.1, qk_norm=norm)
    tol = torch.tensor([24 * n ** 0.5 * 2.0 ** -24 for n in lens], dtype=D, device="cuda")
    each = tol.repeat_interleave(torch.tensor(lens, device="cuda"))[:, None, None]
    info = torch.finfo(dtype)
    fits = (want.abs() < 0.99 * info.max) & (size > 1e-28)
    off = (o.to(D) - want).abs() - info.eps / 2 * want.abs() - info.smallest_normal * info.eps
    assert (~fits | (off <= each * size)).all(), torch.where(fits, off / (each * size), 0.0).max()
    d = (x["state"].to(D) - S).norm(dim=-1)
    assert ((held < 1e-28) | (d <= tol[:, None, None] * held)).all(), (d / (tol[:, None, None] * held)).max()
