"""Filtered sampling against a sorted 64-bit implementation: tokens and kept counts are equal, probabilities are
within fp32's half step (2^-24) and the 64-bit sums' own rounding."""
import numpy as np
import pytest

from delta_ref import sample_row

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    from dfssm_b200 import ops
    return ops


def dev(x, dtype):
    return torch.tensor(np.asarray(x), dtype=dtype, device="cuda")


def run(ops, logits, u, temperature, top_k, top_p, min_p, **kw):
    t, k, p = ops.sample_filtered(logits, dev(u, torch.float32), temperature=dev(temperature, torch.float32),
                                  top_k=dev(top_k, torch.int32), top_p=dev(top_p, torch.float32),
                                  min_p=dev(min_p, torch.float32), **kw)
    return t.tolist(), k.tolist(), p.tolist()


def compare(ops, logits, u, temperature, top_k, top_p, min_p, seen=None, rep=1.0):
    """Every row against the reference; logits a device tensor [B, V]."""
    B, V = logits.shape
    kw = {}
    if seen is not None:
        bits = np.zeros((B, (V + 31) // 32), np.uint32)
        for r, i in zip(*np.nonzero(seen)):
            bits[r, i >> 5] |= np.uint32(1 << (i & 31))
        kw = {"seen_bits": torch.from_numpy(bits.view(np.int32)).cuda(), "rep_penalty": rep}
    got = run(ops, logits, u, temperature, top_k, top_p, min_p, **kw)
    host = logits.float().cpu().numpy()
    for r in range(B):
        want = sample_row(host[r], np.float32(u[r]), np.float32(temperature[r]), int(top_k[r]), np.float32(top_p[r]),
                          np.float32(min_p[r]), None if seen is None else seen[r], rep)
        assert (got[0][r], got[1][r]) == want[:2], (r, got[0][r], got[1][r], want)
        assert abs(got[2][r] - want[2]) <= 2.0 ** -24 * want[2] + 1e-12, (r, got[2][r], want)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 31, 33, 500, 3001, 50281, 151937])
def test_rows_with_settings_of_their_own(ops, V, dtype):
    rng = np.random.default_rng(V)
    B = 12 if V > 10000 else 40
    logits = dev((rng.standard_normal((B, V)) * rng.uniform(0.5, 4, (B, 1))).astype(np.float32), dtype)
    top_k = rng.integers(0, 2, B) * np.exp(rng.uniform(0, np.log(V + 10), B)).astype(np.int64)
    top_p = np.where(rng.random(B) < 0.3, 1.0, rng.uniform(0.05, 0.98, B)).astype(np.float32)
    min_p = np.where(rng.random(B) < 0.5, 0.0, rng.uniform(0, 0.3, B)).astype(np.float32)
    temperature = np.where(rng.random(B) < 0.1, 0.0, rng.uniform(0.3, 1.6, B)).astype(np.float32)
    compare(ops, logits, rng.random(B).astype(np.float32), temperature, top_k, top_p, min_p)


@pytest.mark.parametrize("V", [40, 5000, 60000])
def test_equal_logits_go_to_the_lowest_index(ops, V):
    """Few distinct values, so that every filter ends inside a run of equal logits; -0 and 0 are equal."""
    rng = np.random.default_rng(V)
    B = 24
    logits = rng.integers(-3, 3, (B, V)).astype(np.float32)
    logits[rng.random((B, V)) < 0.2] *= -0.0
    logits[0] = 1.5
    logits[1] = -0.0
    top_k = np.exp(rng.uniform(0, np.log(V), B)).astype(np.int64) * (np.arange(B) % 3 > 0)
    top_p = rng.uniform(0, 1, B).astype(np.float32)
    top_p[0], top_k[0] = 0.3711, 0
    top_p[1], top_k[1] = 0.5001, V // 2
    temperature = np.where(np.arange(B) % 7 == 3, 0, 0.9)
    compare(ops, dev(logits, torch.float32), rng.random(B), temperature, top_k, top_p, np.zeros(B))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [33, 5000, 130000])
def test_masks(ops, V, dtype):
    """-inf, the type's lowest value and NaN in masked places; rows with one token left, and with none."""
    rng = np.random.default_rng(V)
    B = 12
    logits = dev(rng.standard_normal((B, V)).astype(np.float32) * 2, dtype)
    masked = dev(rng.random((B, V)) < 0.9, torch.bool)
    masked[:, V // 2] = False
    masked[5], masked[6], masked[7] = True, True, True
    masked[8] = True
    masked[8, V - 1] = False
    fill = [-np.inf, torch.finfo(dtype).min, np.nan]
    for r in range(B):
        logits[r][masked[r]] = fill[r % 3] if r not in (5, 6) else (-np.inf, np.nan)[r - 5]
    logits[9, V // 2] = np.inf
    logits[10, 3] = logits[10, V - 2] = np.inf
    got = compare(ops, logits, rng.random(B), np.full(B, 1.0), np.full(B, 20) * (np.arange(B) % 2),
                  np.full(B, 0.95), np.full(B, 0.01))
    assert [g[5] for g in got] == [-1, 0, 0] and [g[6] for g in got] == [-1, 0, 0]
    assert got[0][7] >= 0  # all tokens at the lowest finite value: a row of equal logits
    assert got[0][8] == V - 1 and got[2][8] == 1


def test_uniform_at_its_ends(ops):
    """0 takes the first kept token of the vocabulary, anything from the last number below 1 on the last one."""
    logits = np.tile(np.array([[0.0, -np.inf, 1.0, 2.0, -np.inf]], np.float32), (6, 1))
    u = [0.0, 1 - 2.0 ** -24, 1.0, 7.0, -3.0, np.nan]
    got = run(ops, dev(logits, torch.float32), u, [1.0] * 6, [0] * 6, [1.0] * 6, [0.0] * 6)
    assert got[0] == [0, 3, 3, 3, 0, 0] and got[1] == [3] * 6


def test_settings_at_their_ends(ops):
    """top_p 0, negative and NaN, min_p 1 and above, top_k beyond the row, temperatures of 0, below, NaN, tiny, huge."""
    rng = np.random.default_rng(1)
    V = 700
    row = (rng.standard_normal(V) * 3).astype(np.float32)
    rows = [(1, 0, 0.0, 0), (1, 0, -1.0, 0), (1, 0, 1.0, 1.0), (1, 0, 1.0, 5.0), (1, V + 5, 1.0, 0), (1, -4, 1.0, 0),
            (0, 0, 0.9, 0), (-1, 50, 0.9, 0), (np.nan, 50, 0.9, 0), (1e-3, 0, 0.9, 0), (1e4, 0, 0.9, 0), (1, V, 0.9, 0)]
    t, k, p, m = (np.array(c, np.float32) for c in zip(*rows))
    got = compare(ops, dev(np.tile(row, (len(rows), 1)), torch.float32), rng.random(len(rows)), t, k.astype(np.int64), p, m)
    best = int(row.argmax())
    assert all(got[0][i] == best and got[1][i] == 1 for i in (0, 1, 2, 3, 6, 7, 8))
    assert got[1][4] == got[1][5] == V
    nan = run(ops, dev(row[None], torch.float32), [0.5], [1.0], [0], [np.nan], [np.nan])
    assert nan[1] == [V] or nan[1] == [1]


def test_repetition_penalty(ops):
    """Seen tokens' logits are divided whatever their sign, before every filter."""
    rng = np.random.default_rng(4)
    B, V = 8, 1003
    logits = (rng.standard_normal((B, V)) * 4 - 2).astype(np.float32)
    compare(ops, dev(logits, torch.float32), rng.random(B), rng.uniform(0.5, 1.2, B), np.arange(B) * 10,
            np.full(B, 0.9), np.zeros(B), seen=rng.random((B, V)) < 0.2, rep=1.3)


def test_rows_of_a_wider_array_and_defaults(ops):
    """Strided rows, numbers for all rows, no settings at all, and given outputs."""
    rng = np.random.default_rng(5)
    wide = torch.randn(7, 1000, device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    logits, u = wide[:, 13:813], dev(rng.random(7), torch.float32)
    plain = ops.sample_filtered(logits.contiguous(), u)
    out = tuple(torch.full_like(t, 9) for t in plain)
    for got in (ops.sample_filtered(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=out),
                ops.sample_filtered(logits, u, top_k=torch.full((7,), 800, dtype=torch.int32, device="cuda"))):
        assert all(torch.equal(a, b) for a, b in zip(got, plain))
    assert out[1].tolist() == [800] * 7
    assert all(torch.equal(a, b) for a, b in zip(ops.sample_filtered(logits, u, top_k=30, top_p=0.8), (
        ops.sample_filtered(logits.contiguous(), u, top_k=30, top_p=0.8))))
    assert [t.shape[0] for t in ops.sample_filtered(logits[:0], u[:0])] == [0, 0, 0]


def test_draws_follow_the_distribution(ops):
    """20,000 draws of one row, top-k 5: within 5 sigma of the renormalised softmax."""
    n, row = 20000, np.array([1.0, 0.5, 0.0, -0.5, -1.0, 2.0, -3.0], np.float32)
    u = torch.rand(n, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    t, k, _ = ops.sample_filtered(dev(np.tile(row, (n, 1)), torch.float32), u, top_k=5)
    p = np.exp(row.astype(np.float64)) * (np.arange(7) != 4) * (np.arange(7) != 6)
    p /= p.sum()
    c = np.bincount(t.cpu().numpy(), minlength=7)
    assert (k == 5).all() and (np.abs(c - n * p) <= 5 * np.sqrt(n * p * (1 - p))).all()


def test_graph_and_side_stream(ops):
    g = torch.Generator("cuda").manual_seed(8)
    logits, u = torch.randn(33, 50280, device="cuda", generator=g) * 3, torch.rand(33, device="cuda", generator=g)
    kw = {"temperature": torch.full((33,), 0.8, device="cuda"), "top_p": torch.full((33,), 0.9, device="cuda")}
    want = ops.sample_filtered(logits, u, **kw)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        other = ops.sample_filtered(logits, u, **kw)
    out, graph = tuple(torch.empty_like(t) for t in want), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.sample_filtered(logits, u, out=out, **kw)
    for _ in range(2):
        for t in out:
            t.fill_(9)
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, other, out))
