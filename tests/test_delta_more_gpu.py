"""The gated delta rule and filtered sampling at sizes that take other paths of the kernels, and together in a decode
loop.  Tolerances as in test_gated_delta_gpu.py and test_sample_filtered_gpu.py."""
import os
import subprocess
import sys

import numpy as np
import pytest

from delta_ref import sample_row
from helpers import ptr, stream
from test_gated_delta_gpu import args, check, cu, make, reference

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from dfssm_b200 import ops
    return ops


@pytest.mark.parametrize("n_seq", [512, 513, 700])
def test_hundreds_of_sequences(ops, n_seq):
    """More sequences than the chunked kernels put in order; some empty, some without a slot, two on one slot."""
    rng = np.random.default_rng(n_seq)
    heads, lens = (1, 2, 64, 32), rng.integers(0, 12, n_seq)
    lens[7], lens[n_seq - 3] = 150, 70
    x = make(heads, int(lens.sum()), n_seq, torch.float16, 3)
    before = x["state"].clone()
    slots = rng.permutation(n_seq).astype(np.int32)
    lost = [5, 100, n_seq - 1]
    slots[5], slots[100], slots[n_seq - 1] = -1, n_seq, slots[7]
    out = torch.full_like(x["v"], 7.0)
    ops.gated_delta_prefill(*args(x), cu(lens), slots=torch.from_numpy(slots).cuda(), out=out, scale=0.2)
    rows = np.concatenate([[0], np.cumsum(lens)])
    for i in lost:
        assert (out[rows[i]:rows[i + 1]] == 7).all()
    part = [i for i in range(n_seq) if i not in lost]
    own = torch.from_numpy(slots[part].astype(np.int64)).cuda()
    at = torch.from_numpy(np.concatenate([np.arange(rows[i], rows[i + 1]) for i in part])).cuda()
    y = {n: t[at] if n in "qkvab" else t for n, t in x.items()}
    ref = reference(y, lens[part], before[own].cpu().numpy(), 0.2, True)
    check(out[at], x["state"][own], ref, lens[part], torch.float16)
    others = torch.ones(n_seq, dtype=torch.bool, device="cuda")
    others[own] = False
    assert torch.equal(x["state"][others], before[others])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_heads_on_one_key(ops, dtype):
    """Groups of value heads of one key in one block, the last group smaller, over many chunks."""
    x = make((1, 20, 64, 16), 64 * 250 - 9, 1, dtype, 6)
    ref = reference(x, [64 * 250 - 9], x["state"].cpu().numpy(), 0.125, True)
    o = ops.gated_delta_prefill(*args(x), cu([64 * 250 - 9]))
    check(o, x["state"], ref, [64 * 250 - 9], dtype)


@pytest.mark.parametrize("heads", [(2, 4, 128, 128), (1, 40, 128, 64)])
def test_long_sequences_without_a_slot_and_odd_offsets(ops, heads):
    """As the one-token tests of slots and offsets, on lengths that the chunked kernels take."""
    lens = [70, 130, 64, 90]
    x = make(heads, sum(lens), 3, torch.bfloat16, 8)
    before = x["state"].clone()
    out = torch.full_like(x["v"], 7.0)
    ops.gated_delta_prefill(*args(x), cu(lens), slots=torch.tensor([2, 2, -1, 0], dtype=torch.int32, device="cuda"), out=out)
    assert (out[70:264] == 7).all() and torch.equal(x["state"][1], before[1])
    at = torch.cat([torch.arange(70), torch.arange(264, 354)]).cuda()
    y = {n: t[at] if n in "qkvab" else t.clone() for n, t in {**x, "state": before}.items()}
    want = ops.gated_delta_prefill(*args(y), cu([70, 90]), slots=torch.tensor([2, 0], dtype=torch.int32, device="cuda"))
    assert torch.equal(out[at], want) and torch.equal(y["state"], x["state"])
    z = {**x, "state": before.clone()}
    ops.gated_delta_prefill(*args(z), torch.tensor([-5, 70, 30, 999], dtype=torch.int32, device="cuda"))
    assert torch.equal(z["state"][1], before[1]) and torch.isfinite(z["state"]).all()


def test_spoilt_inputs_stay_in_their_sequence(ops):
    lens = [100, 80, 130]
    x = make((1, 4, 128, 64), 310, 3, torch.float16, 12)
    y = {n: t.clone() for n, t in x.items()}
    clean = ops.gated_delta_prefill(*args(x), cu(lens))
    y["k"][120, 0, 5] = float("nan")
    y["v"][150] = float("inf")
    y["q"][179] = float("nan")
    y["a"][160, 2] = float("nan")
    got = ops.gated_delta_prefill(*args(y), cu(lens))
    for i, rows in ((0, slice(0, 100)), (2, slice(180, 310))):
        assert torch.equal(got[rows], clean[rows]) and torch.equal(x["state"][i], y["state"][i])
    assert not torch.isfinite(got[100:180]).all()


def test_first_calls_inside_a_capture():
    """A fresh process whose first call of each op is captured: what the host looks up once must not disturb it."""
    code = """
import sys, torch
sys.path[:0] = [%r, %r]
from dfssm_b200 import ops
from test_gated_delta_gpu import args, cu, make
x = make((1, 4, 128, 64), 200, 2, torch.float16, 1)
y = {n: t.clone() for n, t in x.items()}
logits, u = torch.randn(3, 50280, device="cuda"), torch.rand(3, device="cuda")
p, lens, w = torch.full((3,), 0.9, device="cuda"), cu([130, 70]), torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
o, o1 = torch.empty_like(x["v"]), torch.empty_like(x["v"][:2])
out = (torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, device="cuda"))
one = lambda z: [t[:2] if i < 5 else t for i, t in enumerate(args(z))]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ops.gated_delta_prefill(*args(x), lens, out=o, workspace=w)
    ops.gated_delta_step(*one(x), out=o1)
    ops.sample_filtered(logits, u, top_p=p, out=out)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(o, ops.gated_delta_prefill(*args(y), lens)) and torch.equal(o1, ops.gated_delta_step(*one(y)))
assert torch.equal(x["state"], y["state"])
assert all(torch.equal(a, b) for a, b in zip(out, ops.sample_filtered(logits, u, top_p=p)))
print("same")
""" % (os.path.dirname(os.path.dirname(os.path.abspath(__file__))), os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sampling_beyond_the_lists(ops, dtype):
    """top_k in the thousands and rows of one value: cuts that no short list holds, with one block per row and with
    several, for top-k and top-p."""
    rng = np.random.default_rng(3)
    for B, V in ((3, 50281), (160, 20011), (2, 9000)):
        logits = torch.tensor(rng.standard_normal((B, V)) * 0.3, dtype=dtype, device="cuda")
        logits[0] = 0.25
        logits[1, : V // 2] = -1.0
        k = np.array([rng.integers(2000, V) if r % 2 else 0 for r in range(B)])
        p = rng.uniform(0.3, 0.999, B).astype(np.float32)
        u = rng.random(B).astype(np.float32)
        t, kept, prob = ops.sample_filtered(logits, torch.tensor(u, device="cuda"), top_k=torch.tensor(k, dtype=torch.int32, device="cuda"),
                                            top_p=torch.tensor(p, device="cuda"))
        host = logits.float().cpu().numpy()
        for r in list(range(min(B, 12))):
            want = sample_row(host[r], u[r], 1.0, int(k[r]), p[r])
            assert (t[r].item(), kept[r].item()) == want[:2], (B, V, r, t[r].item(), kept[r].item(), want)
            assert abs(prob[r].item() - want[2]) <= 2.0 ** -24 * want[2] + 1e-12


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompts_then_a_sampled_decode_loop(ops, dtype):
    """A recurrent layer and a language-model head as an engine would run them: ragged prompts through
    gated_delta_prefill, then steps of projection, gated_delta_step, dfssm_lm_head_argmax's logits and sample_filtered,
    each token fed back.  Every recurrence output and state against the token loop on the tensors that were fed, every
    token against the sorted sampler on the logits that were used."""
    from dfssm_b200 import _lib
    lib = _lib.load()
    hk, hv, dk, dv, V, d = 2, 4, 128, 64, 3001, 256
    g = torch.Generator("cuda").manual_seed(1)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    lens, steps = [40, 1, 97], 9
    B, wide = len(lens), 2 * hk * dk + hv * dv + 2 * hv
    emb, proj = randn(V, d).to(dtype), (randn(d, wide) / d ** 0.5).to(dtype)
    A_log, dt_bias = torch.log(1 + 15 * torch.rand(hv, device="cuda", generator=g)), randn(hv) - 4
    Eq = torch.randint(-127, 128, (V, hv * dv), device="cuda", generator=g, dtype=torch.int8)
    Es = torch.full((V,), 0.02, device="cuda")
    state = torch.zeros(B, hv, dv, dk, device="cuda")
    ws = torch.empty(lib.dfssm_lm_head_workspace(B), dtype=torch.uint8, device="cuda")
    fed = [[] for _ in range(B)]  # per sequence: (projection row, o row)

    def layer(tokens):
        y = torch.nn.functional.silu(emb[tokens] @ proj)
        cut = torch.split(y, [hk * dk, hk * dk, hv * dv, hv, hv], 1)
        return y, [cut[0].unflatten(1, (hk, dk)), cut[1].unflatten(1, (hk, dk)), cut[2].unflatten(1, (hv, dv)), cut[3], cut[4],
                   A_log, dt_bias, state]

    prompt = torch.randint(0, V, (sum(lens),), device="cuda", generator=g)
    y, x = layer(prompt)
    o = ops.gated_delta_prefill(*x, cu(lens))
    ends = np.cumsum(lens)
    for i in range(B):
        fed[i] += [(y[r], o[r]) for r in range(ends[i] - lens[i], ends[i])]
    last = o[torch.tensor(ends - 1, device="cuda")]
    kw = dict(temperature=torch.tensor([0.7, 0.0, 1.2], device="cuda"), top_k=torch.tensor([40, 0, 0], dtype=torch.int32, device="cuda"),
              top_p=torch.tensor([0.9, 1.0, 0.8], device="cuda"), min_p=torch.tensor([0.0, 0.0, 0.02], device="cuda"))
    seen = []
    for _ in range(steps):
        logits, best = torch.empty(B, V, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda")
        h = last.reshape(B, hv * dv).half().contiguous()
        _lib.check(lib.dfssm_lm_head_argmax(ptr(Eq), ptr(Es), V, hv * dv, ptr(h), B, ptr(logits), ptr(best), ptr(ws), stream()))
        u = torch.rand(B, device="cuda", generator=g)
        tokens = ops.sample_filtered(logits, u, **kw)[0]
        seen.append((logits, u, tokens))
        y, x = layer(tokens.long())
        last = ops.gated_delta_step(*x)
        for i in range(B):
            fed[i].append((y[i], last[i]))
    rows = torch.stack([r for f in fed for r, _ in f])
    cut = torch.split(rows, [hk * dk, hk * dk, hv * dv, hv, hv], 1)
    z = {"q": cut[0].unflatten(1, (hk, dk)), "k": cut[1].unflatten(1, (hk, dk)), "v": cut[2].unflatten(1, (hv, dv)), "a": cut[3], "b": cut[4],
         "A_log": A_log, "dt_bias": dt_bias}
    n = [m + steps for m in lens]
    ref = reference(z, n, np.zeros(state.shape), dk ** -0.5, True)
    check(torch.stack([w for f in fed for _, w in f]), state, ref, n, dtype)
    for logits, u, tokens in seen:
        for i in range(B):
            want = sample_row(logits[i].cpu().numpy(), u[i].item(), *(float(kw[s][i]) if s != "top_k" else int(kw[s][i])
                                                                    for s in ("temperature", "top_k", "top_p", "min_p")))
            assert tokens[i].item() == want[0]


def test_model_samples_from_its_logits():
    """DFSSMModel.sample: the logits of forward(), filtered, and the tokens fed back."""
    from helpers import model, weights
    m = model(weights("tiny"), 3)
    m.reset_state()
    u = torch.tensor([0.1, 0.5, 0.9], device="cuda")
    logits = m.forward(torch.tensor([1, 2, 3])).clone()
    tokens = m.sample(u, temperature=0.8, top_k=20, top_p=0.9)
    for i in range(3):
        assert tokens[i].item() == sample_row(logits[i].cpu().numpy(), u[i].item(), np.float32(0.8), 20, np.float32(0.9))[0]
    assert torch.equal(m.sample(u, temperature=0.0), logits.argmax(-1).int())
    m.step(tokens)
    m.close()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens", [[150], [5]])
def test_decays_of_the_largest_gates(ops, lens, dtype):
    """a at the type's largest value and at infinity: that token forgets everything before it, and the tokens after it
    decay by gates of their own, in every form of the op."""
    heads = (1, 4, 128, 32)
    x = make(heads, lens[0], 1, dtype, 21)
    x["a"][2::9, 0] = torch.finfo(dtype).max
    x["a"][1::70, 1] = float("inf")
    x["a"][3::20, 2] = float("inf")
    x["a"][::2, 3] = -torch.finfo(dtype).max
    x["a"][1, 3] = float("-inf")
    ref = reference(x, lens, x["state"].cpu().numpy(), 0.3, True)
    o = ops.gated_delta_prefill(*args(x), cu(lens), scale=0.3)
    check(o, x["state"], ref, lens, dtype)


@pytest.mark.parametrize("shape", ["bulk", "coarse", "crowded", "far"])
@pytest.mark.parametrize("B,V", [(9, 50281), (150, 6000)])
def test_lists_of_every_length(ops, B, V, shape):
    """top_k around every way a short list is ordered (by one warp, by counting, in buckets, in crowded ones), over
    spread, equal and crowded logits, alone and with top-p and min-p that keep few or many of the list."""
    rng = np.random.default_rng(len(shape) + B)
    logits = (rng.standard_normal((B, V)) * 1.5).astype(np.float32)
    if shape == "coarse":
        logits = np.round(logits * 4) / 4  # dozens of equal ones at the cut
    elif shape == "crowded":
        logits = 3 + 1e-3 * logits
        logits[:, 17] = 12.0  # the rest shares one bucket
    elif shape == "far":
        logits[:, 5] = 250.0
        logits[::2, ::3] = -3e38
    sizes = np.array([2, 31, 64, 65, 130, 257, 900, 1025, 2048])
    k = sizes[np.arange(B) % len(sizes)]
    u = rng.random(B).astype(np.float32)
    dev = {"u": torch.tensor(u, device="cuda"), "logits": torch.tensor(logits, device="cuda")}
    for top_p, min_p in ((None, None), (0.5, None), (0.97, 0.001), (None, 0.1)):
        t, kept, prob = ops.sample_filtered(dev["logits"], dev["u"], top_k=torch.tensor(k, dtype=torch.int32, device="cuda"),
                                            top_p=top_p, min_p=min_p)
        for r in range(min(B, 27)):
            want = sample_row(logits[r], u[r], 1.0, int(k[r]), 1.0 if top_p is None else top_p, min_p or 0.0)
            assert (t[r].item(), kept[r].item()) == want[:2], (r, k[r], top_p, min_p, t[r].item(), kept[r].item(), want)
            assert abs(prob[r].item() - want[2]) <= 2.0 ** -24 * want[2] + 1e-12


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(2, 4, 128, 128), (1, 3, 64, 48)])
def test_decode_rows_and_prompts_in_one_call(ops, heads, dtype):
    """One-token rows, short and long prompts, empty ones and padding together: the kernels share them by length."""
    rng = np.random.default_rng(heads[3])
    lens = np.array([1] * 40 + [12] * 9 + [13] * 7 + [300, 65, 64, 2] + [0] * 3)
    rng.shuffle(lens)
    n_seq, n = len(lens), int(lens.sum())
    x = make(heads, n + 5, n_seq + 2, dtype, 31)
    slots = rng.permutation(n_seq + 2)[:n_seq].astype(np.int32)
    lost = [int(np.flatnonzero(lens == m)[-1]) for m in (1, 13)]
    slots[lost[0]], slots[lost[1]] = -1, slots[int(np.flatnonzero(lens == 12)[0])]
    lost = [i for i in range(n_seq) if slots[i] < 0 or slots[i] in slots[:i]]
    before, out = x["state"].clone(), torch.full_like(x["v"], 7.0)
    ops.gated_delta_prefill(*args(x), cu(lens), slots=torch.from_numpy(slots).cuda(), out=out, scale=0.2)
    rows = np.concatenate([[0], np.cumsum(lens)])
    assert (out[n:] == 7).all() and all((out[rows[i]:rows[i + 1]] == 7).all() for i in lost)
    part = [i for i in range(n_seq) if i not in lost]
    own = torch.from_numpy(slots[part].astype(np.int64)).cuda()
    at = torch.from_numpy(np.concatenate([np.arange(rows[i], rows[i + 1]) for i in part])).cuda()
    y = {m: t[at] if m in "qkvab" else t for m, t in x.items()}
    ref = reference(y, lens[part], before[own].cpu().numpy(), 0.2, True)
    check(out[at], x["state"][own], ref, lens[part], dtype)
    others = torch.ones(n_seq + 2, dtype=torch.bool, device="cuda")
    others[own] = False
    assert torch.equal(x["state"][others], before[others])


@pytest.mark.parametrize("B", [300, 1025, 4096, 4097])
def test_more_rows_than_run_at_once(ops, B):
    """Batches whose rows are taken in another order than their own, with settings of all kinds."""
    rng = np.random.default_rng(B)
    V = 600
    logits = (rng.standard_normal((B, V)) * 2).astype(np.float32)
    u = rng.random(B).astype(np.float32)
    kind = rng.integers(0, 5, B)
    k = np.where(kind < 2, 0, rng.integers(1, 200, B)).astype(np.int32)
    p = np.where((kind == 1) | (kind == 2), 1.0, rng.uniform(0.3, 0.99, B)).astype(np.float32)
    t = np.where(kind == 4, 0.0, rng.uniform(0.5, 1.5, B)).astype(np.float32)
    dev = lambda x: torch.tensor(x, device="cuda")  # noqa: E731
    token, kept, prob = ops.sample_filtered(dev(logits), dev(u), temperature=dev(t), top_k=dev(k), top_p=dev(p))
    token, kept, prob = token.tolist(), kept.tolist(), prob.tolist()
    for r in rng.permutation(B)[:400]:
        want = sample_row(logits[r], u[r], t[r], int(k[r]), p[r])
        assert (token[r], kept[r]) == want[:2], (r, kind[r], token[r], kept[r], want)
        assert abs(prob[r] - want[2]) <= 2.0 ** -24 * want[2] + 1e-12
    assert min(token) >= 0 and max(token) < V  # every row was taken
