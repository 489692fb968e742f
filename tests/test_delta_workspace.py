"""The prompt op's workspace: no larger than what the chunks of a call can use, and no byte behind it touched."""
import numpy as np
import pytest

from dfssm_b200 import _lib

CHUNK_BYTES = 22 * 1024  # of one chunk and value head, at most


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.parametrize("tokens,n_seq", [(600, 600), (256, 256), (2047, 512), (512, 512), (5, 5), (12, 3), (800, 40), (40, 2), (1, 1)])
def test_workspace_of_short_sequences(lib, tokens, n_seq):
    """Sequences that the token loop takes (up to 12 tokens) need no chunks, and calls of nothing else no workspace to speak of."""
    need = lib.dfssm_gated_delta_workspace(tokens, n_seq, 1, 64, 128, 64, 0)
    if tokens <= 12:
        assert need <= 4096
    assert need <= (tokens // 64 + tokens // 13 + 1) * 64 * CHUNK_BYTES + 16 * n_seq


def test_workspace_of_long_sequences(lib):
    for tokens, n_seq in ((32768, 1), (16384, 24), (4096, 64)):
        need = lib.dfssm_gated_delta_workspace(tokens, n_seq, 16, 32, 128, 128, 0)
        assert tokens // 64 * 32 * 20480 <= need <= (tokens // 64 + n_seq) * 32 * CHUNK_BYTES + 16 * n_seq


def test_a_workspace_for_the_largest_call_is_enough_for_smaller_ones(lib):
    """More tokens or more sequences never need less."""
    sizes = [1, 2, 12, 13, 31, 32, 33, 64, 200, 511, 512, 513, 600, 1023, 1024, 2047, 2048, 5000, 16384, 16385]
    need = [[lib.dfssm_gated_delta_workspace(t, n, 2, 4, 128, 64, 1) for n in sizes] for t in sizes]
    assert all(a <= b for row in need for a, b in zip(row, row[1:])) and all(a <= b for col in zip(*need) for a, b in zip(col, col[1:]))


def test_chunk_numbers_are_distinct():
    """The numbering by rows that the smaller workspace rests on: cu / 64 + cu / 13 + c for sequences of 13 tokens and more."""
    rng = np.random.default_rng(0)
    for _ in range(300):
        lens = rng.choice([0, 1, 12, 13, 14, 25, 26, 63, 64, 65, 77, 128, 129, 500], rng.integers(1, 60))
        cu, seen = np.concatenate([[0], np.cumsum(lens)]), -1
        for first, n in zip(cu, lens):
            if n >= 13:
                base = first // 64 + first // 13
                assert base > seen
                seen = base + (n + 63) // 64 - 1
        assert seen <= cu[-1] // 64 + cu[-1] // 13


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("lens", [[1] * 300 + [13] * 4 + [70] + [1] * 50, [12] * 20 + [13] * 20 + [14] * 3, [1, 40], [1] * 500 + [600], [3, 4]],
                         ids=lambda v: "%d in %d" % (sum(v), len(v)))
def test_nothing_behind_the_workspace(lib, lens, dtype):
    import torch
    from dfssm_b200 import ops
    from test_gated_delta_gpu import args, check, cu, make, reference
    heads, t = (1, 3, 128, 32), getattr(torch, dtype)
    lens = np.random.default_rng(len(lens)).permutation(lens).tolist()
    x = make(heads, sum(lens), len(lens), t, 5)
    need = ops.gated_delta_workspace(sum(lens), len(lens), *heads, t)
    room = torch.full((need + 8192,), 171, dtype=torch.uint8, device="cuda")
    ref = reference(x, lens, x["state"].cpu().numpy(), 0.1, True)
    o = ops.gated_delta_prefill(*args(x), cu(lens), scale=0.1, workspace=room[:need])
    check(o, x["state"], ref, lens, t)
    assert (room[need:] == 171).all()


def test_many_sequences_have_chunks(lib):
    """However many sequences there are, a long prompt among one-token rows is not left to the token loop: its chunks have a place."""
    for tokens, n_seq in ((599 + 1700, 600), (2000, 1000), (100000, 30000)):
        assert lib.dfssm_gated_delta_workspace(tokens, n_seq, 1, 64, 128, 64, 0) >= (tokens // 64) * 64 * 20480


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("named", [False, True], ids=["slots in order", "slots"])
@pytest.mark.parametrize("lens", [[1] * 599 + [700], [1] * 700 + [0] * 30 + [13] * 9 + [12] * 9 + [300, 65], [1] * 700 + [14] * 600 + [200]],
                         ids=lambda v: "%d in %d" % (sum(v), len(v)))
def test_prompts_among_hundreds_of_rows(lens, named, dtype):
    """More than 512 sequences with long ones among them; 601 long ones in the last case.  Some without a slot, some twice."""
    import torch
    from dfssm_b200 import ops
    from test_gated_delta_gpu import args, check, cu, make, reference
    heads, t, rng = (1, 2, 64, 32), getattr(torch, dtype), np.random.default_rng(len(lens))
    lens = rng.permutation(lens)
    n_seq, n = len(lens), int(lens.sum())
    x = make(heads, n + 3, n_seq, t, 6)
    slots, lost = np.arange(n_seq), []
    if named:
        slots = rng.permutation(n_seq)
        longest, one = int(lens.argmax()), int(np.flatnonzero(lens == 1)[-1])
        slots[one] = -1
        slots[int(np.flatnonzero(lens == lens[lens > 1].min())[0])] = n_seq
        if longest:
            slots[longest - 1 if longest > 1 else 0] = slots[longest]  # of two on one slot the earlier one has it
        lost = [i for i in range(n_seq) if not 0 <= slots[i] < n_seq or slots[i] in slots[:i]]
    before, out = x["state"].clone(), torch.full_like(x["v"], 7.0)
    ops.gated_delta_prefill(*args(x), cu(lens), out=out, scale=0.2,
                            slots=torch.tensor(slots, dtype=torch.int32, device="cuda") if named else None)
    rows = np.concatenate([[0], np.cumsum(lens)])
    assert (out[n:] == 7).all() and all((out[rows[i]:rows[i + 1]] == 7).all() for i in lost)
    part = [i for i in range(n_seq) if i not in set(lost)]
    own = torch.tensor(slots[part], device="cuda")
    at = torch.from_numpy(np.concatenate([np.arange(rows[i], rows[i + 1]) for i in part])).cuda()
    y = {m: v[at] if m in "qkvab" else v for m, v in x.items()}
    ref = reference(y, lens[part], before[own].cpu().numpy(), 0.2, True)
    check(out[at], x["state"][own], ref, lens[part], t)
    others = torch.ones(n_seq, dtype=torch.bool, device="cuda")
    others[own] = False
    assert torch.equal(x["state"][others], before[others])
