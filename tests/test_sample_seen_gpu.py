"""The repetition penalty of filtered sampling wherever a row's x comes from: one block or a cluster per row, its slice in shared
memory or computed again from the logits in every pass, aligned rows or not, 32 and 16 bits.  Tolerances as in
test_sample_filtered_gpu.py."""
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


def packed(seen):
    B, V = seen.shape
    wide = np.zeros((B, (V + 31) // 32 * 32), bool)
    wide[:, :V] = seen
    return torch.from_numpy(np.packbits(wide, axis=1, bitorder="little").view(np.int32)).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("apart", [0, 3], ids=["contiguous", "strided"])
@pytest.mark.parametrize("B,V", [(3, 33), (200, 33), (3, 5000), (200, 5000), (3, 50281), (170, 50281), (2, 151937), (150, 151937)])
def test_seen_tokens(ops, B, V, apart, dtype):
    rng = np.random.default_rng(B + V + apart)
    g = torch.Generator("cuda").manual_seed(B + V)
    room = torch.randn(B, V + apart, device="cuda", generator=g).mul_(3).to(dtype)
    logits = room[:, apart:]  # with apart, rows that start at odd places
    few = min(B, 12)
    seen = np.zeros((B, V), bool)
    seen[:few] = rng.random((few, V)) < rng.choice([0.01, 0.3, 0.99], (few, 1))
    host = logits[:few].float().cpu().numpy()
    best = np.argsort(-host, axis=1)[:, : max(1, V // 50)]
    np.put_along_axis(seen[:few], best, rng.random(best.shape) < 0.5, 1)  # among those that would be drawn too
    seen[0], seen[1] = True, False
    top_k = np.where(rng.random(B) < 0.5, 0, np.exp(rng.uniform(0, np.log(V), B))).astype(np.int32)
    top_p = np.where(rng.random(B) < 0.3, 1.0, rng.uniform(0.2, 0.99, B)).astype(np.float32)
    min_p = np.where(rng.random(B) < 0.5, 0.0, rng.uniform(0, 0.2, B)).astype(np.float32)
    temperature = np.where(rng.random(B) < 0.15, 0.0, rng.uniform(0.4, 1.5, B)).astype(np.float32)
    top_k[1] = 0  # a whole row without a list
    u = rng.random(B).astype(np.float32)
    rep = 1.35
    dev = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    token, kept, prob = ops.sample_filtered(logits, dev(u), temperature=dev(temperature), top_k=dev(top_k), top_p=dev(top_p),
                                            min_p=dev(min_p), seen_bits=packed(seen), rep_penalty=rep)
    token, kept, prob = token.tolist(), kept.tolist(), prob.tolist()
    for r in range(few):
        want = sample_row(host[r], u[r], temperature[r], int(top_k[r]), top_p[r], min_p[r], seen[r], rep)
        assert (token[r], kept[r]) == want[:2], (r, top_k[r], top_p[r], min_p[r], temperature[r], token[r], kept[r], want)
        assert abs(prob[r] - want[2]) <= 2.0 ** -24 * want[2] + 1e-12, (r, prob[r], want)


def test_a_penalty_of_one_changes_nothing(ops):
    g = torch.Generator("cuda").manual_seed(4)
    logits, u = torch.randn(40, 60001, device="cuda", generator=g), torch.rand(40, device="cuda", generator=g)
    bits = torch.randint(-2 ** 31, 2 ** 31 - 1, (40, (60001 + 31) // 32), device="cuda", generator=g).int()
    plain = ops.sample_filtered(logits, u, top_p=0.9)
    assert all(torch.equal(a, b) for a, b in zip(plain, ops.sample_filtered(logits, u, top_p=0.9, seen_bits=bits, rep_penalty=1.0)))
