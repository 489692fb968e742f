"""The gated delta rule ops against a 64-bit token loop.

Tolerances.  A token's update rounds S k (a sum of dk products in fp32), the decay (expf of a gate of a few
fp32 roundings), beta, u and the new state, at most 24 half steps of fp32 (2^-24) of the row's size in all;
independent roundings of T tokens add up in quadrature, so a state is within 24 sqrt(T) 2^-24 of the size it
has or still remembers, and o within the same share of scale |S_r| |q|, plus half a step of its own type.
(Products with operands split into two fp16 parts are off by 2^-22 of the product, four of the half steps.)
"""
import numpy as np
import pytest

from delta_ref import delta_rule

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

HEADS = [(1, 3, 128, 64), (2, 4, 128, 128), (2, 2, 64, 64), (1, 2, 128, 16), (1, 1, 64, 256), (3, 6, 128, 48)]
TYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    from dfssm_b200 import ops
    return ops


def make(heads, n, n_slots, dtype, seed, norm=True, spread=1.0):
    hk, hv, dk, dv = heads
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    silu = torch.nn.functional.silu
    q, k, v = silu(r(n, hk, dk)), silu(r(n, hk, dk)), spread * silu(r(n, hv, dv))
    if not norm:
        q, k = (x / x.norm(dim=-1, keepdim=True).clamp_min(1e-3) for x in (q, k))
    x = {"q": q, "k": k, "v": v, "a": r(n, hv), "b": r(n, hv)}
    x = {name: t.to(dtype).cuda() for name, t in x.items()}
    x["A_log"] = torch.log(1 + 15 * torch.rand(hv, generator=g)).cuda()
    dt = torch.exp(torch.rand(hv, generator=g) * 4.6 - 6.9)
    x["dt_bias"] = (dt + torch.log(-torch.expm1(-dt))).cuda()
    x["state"] = (0.3 * spread * r(n_slots, hv, dv, dk)).cuda()
    return x


def reference(x, lens, starts, scale, norm):
    h = {name: t.double().cpu().numpy() for name, t in x.items()}
    return delta_rule(h["q"], h["k"], h["v"], h["a"], h["b"], h["A_log"], h["dt_bias"], starts, lens, scale, norm)


def check(o, state, ref, lens, dtype, scale=None):
    ro, rS, size, held = ref
    at = 0
    for i, n in enumerate(lens):
        tol = 24 * np.sqrt(max(n, 1)) * 2.0 ** -24
        got, want = o[at:at + n].double().cpu().numpy(), ro[at:at + n]
        off = np.abs(got - want) - torch.finfo(dtype).eps / 2 * np.abs(want) - tol * size[at:at + n]
        assert (off <= torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all(), (i, n, off.max())
        d = np.sqrt(((state[i].double().cpu().numpy() - rS[i]) ** 2).sum((-1, -2)))
        assert (d <= tol * held[i]).all(), (i, n, (d / (2.0 ** -24 * held[i])).max())
        at += n


def args(x):
    return [x[n] for n in ("q", "k", "v", "a", "b", "A_log", "dt_bias", "state")]


def cu(lens, first=0):
    return torch.tensor(first + np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("B", [1, 5])
def test_step(ops, heads, B, norm, dtype):
    x = make(heads, B, B + 2, dtype, 7 * B, norm)
    slots = torch.tensor(np.random.default_rng(B).permutation(B + 2)[:B].astype(np.int32), device="cuda")
    before = x["state"].clone()
    scale = heads[2] ** -0.5
    ref = reference(x, [1] * B, before[slots.long()].cpu().numpy(), scale, norm)
    o = ops.gated_delta_step(*args(x), slots=slots, qk_norm=norm)
    check(o, x["state"][slots.long()], ref, [1] * B, dtype)
    others = torch.ones(B + 2, dtype=torch.bool, device="cuda")
    others[slots.long()] = False
    assert torch.equal(x["state"][others], before[others])


LENS = [[1], [16], [0, 1, 63, 64, 65], [2, 0, 130, 7], [200], [1] * 9 + [33], [129, 128, 127]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens", LENS, ids=lambda v: "-".join(map(str, v)))
def test_prefill(ops, heads, lens, dtype):
    norm = len(lens) != 4
    n, n_seq = sum(lens), len(lens)
    x = make(heads, n, n_seq + 1, dtype, n + heads[1], norm)
    slots = torch.tensor(np.random.default_rng(n).permutation(n_seq + 1)[:n_seq].astype(np.int32), device="cuda")
    before = x["state"].clone()
    ref = reference(x, lens, before[slots.long()].cpu().numpy(), 0.11, norm)
    o = ops.gated_delta_prefill(*args(x), cu(lens), slots=slots, scale=0.11, qk_norm=norm)
    check(o, x["state"][slots.long()], ref, lens, dtype)
    other = (set(range(n_seq + 1)) - set(slots.tolist())).pop()
    assert torch.equal(x["state"][other], before[other])
    assert torch.equal(x["state"][slots.long()][[i for i, m in enumerate(lens) if m == 0]],
                       before[slots.long()][[i for i, m in enumerate(lens) if m == 0]])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[70], [3]])
def test_gates_at_their_ends(ops, lens, dtype):
    """Decays down to e^-1000 and to almost none, beta of 0 and 1, keys and queries of zero, values of 1e4:
    the state may vanish and come back within a chunk."""
    n, heads = sum(lens), (1, 4, 128, 32)
    x = make(heads, n, 1, dtype, 3)
    x["a"][:, 0] = 60.0  # |g| up to 1000 a token
    x["a"][:, 1] = -30.0  # g = 0
    x["a"][::3, 2] = 60.0
    x["b"][:, 1] = 30.0
    x["b"][::2, 2] = -30.0
    x["k"][::4] = 0
    x["q"][::5] = 0
    x["v"][1::7] *= 1e4
    ref = reference(x, lens, x["state"].cpu().numpy(), 1.0, True)
    o = ops.gated_delta_prefill(*args(x), cu(lens), scale=1.0)
    check(o, x["state"], ref, lens, dtype)
    assert torch.isfinite(x["state"]).all() and torch.isfinite(o).all()


def test_parallel_keys(ops):
    """One key for all tokens of a long chunk, beta near 1: the triangular system is as far from diagonal as it gets."""
    x = make((1, 2, 128, 64), 150, 1, torch.float16, 5)
    x["k"][:] = x["k"][0]
    x["b"][:] = 6.0
    x["a"][:] = -8.0
    ref = reference(x, [150], x["state"].cpu().numpy(), 1.0, True)
    o = ops.gated_delta_prefill(*args(x), cu([150]), scale=1.0)
    check(o, x["state"], ref, [150], torch.float16)


@pytest.mark.parametrize("dtype", TYPES)
def test_views_of_one_projection(ops, dtype):
    """q, k and v as column ranges of one wide row, o into a wide row, as a decode loop has them; rows of o behind
    the last sequence and columns beside the range stay as they were."""
    hk, hv, dk, dv = 2, 4, 128, 64
    lens, n = [90, 5], 100
    x = make((hk, hv, dk, dv), n, 2, dtype, 11)
    wide = torch.zeros(n, 2 * hk * dk + hv * dv + 24, dtype=dtype, device="cuda")
    cut = {"q": (8, hk, dk), "k": (8 + hk * dk, hk, dk), "v": (16 + 2 * hk * dk, hv, dv)}
    y = dict(x)
    for name, (c, h, d) in cut.items():
        y[name] = wide[:, c:c + h * d].unflatten(1, (h, d))
        y[name].copy_(x[name])
    gates = torch.stack([x["a"], x["b"]], 1)  # [n, 2, hv]
    y["a"], y["b"] = gates[:, 0], gates[:, 1]
    x["state"], y["state"] = x["state"].clone(), x["state"].clone()
    room = torch.full((n, hv * dv + 16), 7.0, dtype=dtype, device="cuda")
    out = room[:, 8:8 + hv * dv].unflatten(1, (hv, dv))
    ops.gated_delta_prefill(*args(x), cu(lens), out=(plain := torch.full_like(x["v"], 7.0)))
    ops.gated_delta_prefill(*args(y), cu(lens), out=out)
    assert torch.equal(out, plain) and torch.equal(x["state"], y["state"])
    assert (room[:, :8] == 7).all() and (room[:, 8 + hv * dv:] == 7).all() and (plain[95:] == 7).all()


@pytest.mark.parametrize("op", ["step", "prefill"])
def test_slots_that_take_no_part(ops, op):
    """Slots out of range, and the second of two equal ones, leave state and rows of o as they were."""
    heads, n = (1, 2, 128, 32), 5
    x = make(heads, n, 4, torch.float16, 2)
    before = x["state"].clone()
    slots = torch.tensor([2, -1, 2, 4, 0], dtype=torch.int32, device="cuda")
    out = torch.full_like(x["v"], 7.0)
    if op == "step":
        ops.gated_delta_step(*args(x), slots=slots, out=out)
    else:
        ops.gated_delta_prefill(*args(x), cu([1] * 5), slots=slots, out=out)
    y = {**x, "state": before.clone()}
    want = ops.gated_delta_step(*[t[[0, 4]] if i < 5 else t for i, t in enumerate(args(y))],
                                slots=torch.tensor([2, 0], dtype=torch.int32, device="cuda"))
    assert torch.equal(out[[0, 4]], want) and (out[1:4] == 7).all()
    assert torch.equal(x["state"], y["state"])


def test_offsets_that_do_not_fit(ops):
    """Offsets below 0, beyond the rows or falling are clamped: nothing else is read or written."""
    x = make((1, 2, 128, 32), 10, 3, torch.float16, 2)
    before = x["state"].clone()
    out = torch.full_like(x["v"], 7.0)
    bad = torch.tensor([-5, 4, 3, 99], dtype=torch.int32, device="cuda")  # tokens 0..3, none, 3..9
    ops.gated_delta_prefill(*args(x), bad, out=out)
    assert torch.equal(x["state"][1], before[1]) and torch.isfinite(out).all()
    y = {**x, "state": before.clone()}
    ops.gated_delta_prefill(*args(y), torch.tensor([3, 3, 3, 10], dtype=torch.int32, device="cuda"))
    assert torch.equal(x["state"][2], y["state"][2])


def test_nothing_to_do(ops):
    x = make((1, 2, 128, 32), 3, 2, torch.float16, 2)
    before = x["state"].clone()
    none = [t[:0] if i < 5 else t for i, t in enumerate(args(x))]
    assert ops.gated_delta_step(*none).shape == (0, 2, 32)
    assert ops.gated_delta_prefill(*none, cu([0, 0])).shape == (0, 2, 32)
    assert ops.gated_delta_prefill(*args(x), cu([])).shape == (3, 2, 32)
    assert torch.equal(x["state"], before)


@pytest.mark.parametrize("lens", [[65, 30], [300]])
def test_prefill_then_steps_is_one_prefill(ops, lens):
    """A prompt in one call, and in two calls with single tokens between them, on the 1.3B shape's heads."""
    heads, n = (1, 64, 128, 64), sum(lens)
    x = make(heads, n, len(lens), torch.float16, 1)
    start = x["state"].clone()
    o = ops.gated_delta_prefill(*args(x), cu(lens))
    rows = cu(lens).tolist()
    y = {**x, "state": start.clone()}
    ends = [20, 25]  # every sequence: 20 tokens, 5 steps, the rest
    pick = lambda lo, hi: torch.cat([torch.arange(r + lo, min(r + hi, rows[i + 1])) for i, r in enumerate(rows[:-1])]).cuda()  # noqa: E731
    part = lambda at: [t[at] if i < 5 else t for i, t in enumerate(args(y))]  # noqa: E731
    got = torch.empty_like(o)
    at = pick(0, 20)
    got[at] = ops.gated_delta_prefill(*part(at), cu([20] * len(lens)))
    for s in range(*ends):
        at = pick(s, s + 1)
        got[at] = ops.gated_delta_step(*part(at))
    at = pick(25, 10 ** 6)
    got[at] = ops.gated_delta_prefill(*part(at), cu([m - 25 for m in lens]))
    tol = 2 * 24 * np.sqrt(max(lens)) * 2.0 ** -24
    assert ((y["state"] - x["state"]).norm() <= tol * x["state"].norm()).item()
    d = (got.float() - o.float()).abs()
    assert (d <= 2.0 ** -10 * o.float().abs() + tol * o.float().abs().max() * 12).all()


def test_streams_graphs_and_workspaces(ops):
    """Two streams at once, each with its own workspace, and a captured graph replayed: the bits of a plain call."""
    heads, lens = (2, 4, 128, 128), [200, 70, 1]
    x = make(heads, sum(lens), 3, torch.bfloat16, 4)
    start, offsets = x["state"].clone(), cu(lens)
    want = ops.gated_delta_prefill(*args(x), offsets)
    state1 = x["state"].clone()
    want2 = ops.gated_delta_step(*[t[:3] if i < 5 else t for i, t in enumerate(args(x))])
    state2 = x["state"].clone()
    bytes_ = ops.gated_delta_workspace(sum(lens), 3, *heads, torch.bfloat16)
    runs = []
    torch.cuda.synchronize()
    for _ in range(2):
        y, s = {**x, "state": start.clone()}, torch.cuda.Stream()
        w = torch.empty(bytes_, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            runs.append((ops.gated_delta_prefill(*args(y), offsets, workspace=w), y["state"], w))
    torch.cuda.synchronize()
    for o, state, _ in runs:
        assert torch.equal(o, want) and torch.equal(state, state1)
    y, out, out2 = {**x, "state": start.clone()}, torch.empty_like(want), torch.empty_like(want2)
    w, graph = torch.empty(bytes_, dtype=torch.uint8, device="cuda"), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.gated_delta_prefill(*args(y), offsets, out=out, workspace=w)
        ops.gated_delta_step(*[t[:3] if i < 5 else t for i, t in enumerate(args(y))], out=out2)
    for _ in range(2):
        y["state"].copy_(start)
        w.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2, want2) and torch.equal(y["state"], state2)


def test_offsets_past_32_bits(ops):
    """State slots and token rows more than 2^31 elements from the start of their arrays."""
    heads = (1, 64, 128, 64)
    slots = 2 ** 31 // (64 * 64 * 128) + 2
    x = make(heads, 70, 1, torch.float16, 9)
    small = x["state"].clone()
    want = ops.gated_delta_prefill(*args(x), cu([70]))
    big = torch.empty(slots, *small.shape[1:], device="cuda")
    big[-1] = small[0]
    ld = 8192
    rows = 2 ** 31 // ld + 80
    room = torch.empty(rows, ld, dtype=torch.float16, device="cuda")
    v = room[:, :4096].unflatten(1, (64, 64))
    q, k = (room[:, c:c + 128].unflatten(1, (1, 128)) for c in (4096, 4224))
    a, b = room[:, 4352:4416], room[:, 4416:4480]
    for to, name in ((q, "q"), (k, "k"), (v, "v"), (a, "a"), (b, "b")):
        to[-70:] = x[name]
    o = torch.empty(rows, ld, dtype=torch.float16, device="cuda")[:, :4096].unflatten(1, (64, 64))
    last = torch.tensor([slots - 1], dtype=torch.int32, device="cuda")
    ops.gated_delta_prefill(q, k, v, a, b, x["A_log"], x["dt_bias"], big, cu([70], rows - 70), slots=last, out=o)
    assert torch.equal(o[-70:], want) and torch.equal(big[-1], x["state"][0])
    o1 = ops.gated_delta_step(*[t[:1] if i < 5 else t for i, t in enumerate(args(x))])
    o2 = ops.gated_delta_step(*[t[:1] if i < 5 else t for i, t in enumerate(args({**x, "state": big}))], slots=last)
    assert torch.equal(o1, o2) and torch.equal(big[-1], x["state"][0])
