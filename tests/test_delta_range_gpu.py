"""The gated delta rule over inputs whose sizes lie far apart: what a sequence has forgotten, or does not know yet, must not
cost the tokens beside it their bits.  Tolerances as in test_gated_delta_gpu.py: of the size that a head's state has or
still remembers at each token."""
import numpy as np
import pytest

from test_gated_delta_gpu import args, check, cu, make, reference

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# heads for walks whose blocks all have an SM, and for walks of two blocks per SM
HEADS = [(1, 2, 128, 32), (2, 4, 64, 48), (2, 40, 128, 128)]
SIZES = [(torch.float16, 3e4, 1e-2), (torch.float16, 6e4, 1e-3), (torch.float16, 6e4, 6e-5), (torch.bfloat16, 1e8, 1.0),
         (torch.bfloat16, 1e10, 1.0), (torch.bfloat16, 1e13, 1.0)]
FORGET = 60.0  # a gate of |g| > 60: e^g leaves nothing


@pytest.fixture(scope="module")
def ops():
    from dfssm_b200 import ops
    return ops


def far_apart(heads, lens, dtype, big, small, mode, seed=1):
    """Values of `small`, and of `big` where the mode says; gates that keep, but for those that forget."""
    x = make(heads, sum(lens), len(lens), torch.float32, seed)
    x["a"][:] = -8.0
    x["v"] *= small
    x["state"] *= small
    starts = np.concatenate([[0], np.cumsum(lens)])[:-1]
    for at, n in zip(starts, lens):
        for t in range(at + 10, at + n - 2, 64):  # once in every chunk
            if mode in ("value then gate", "value, gate, value"):
                x["v"][t] *= big / small
                x["a"][t + 1] = FORGET
            if mode in ("small before big", "value, gate, value") and t + 25 < at + n:
                x["v"][t + 25] *= big / small
        if mode == "old state":
            x["a"][at + 3] = FORGET
    if mode == "old state":
        x["state"] *= big / small
    lim = torch.finfo(dtype).max
    return {name: t.clamp(-lim, lim).to(dtype) if name in "qkvab" else t for name, t in x.items()}


@pytest.mark.parametrize("mode", ["value then gate", "value, gate, value", "small before big", "old state"])
@pytest.mark.parametrize("dtype,big,small", SIZES, ids=lambda v: str(v).replace("torch.", ""))
@pytest.mark.parametrize("heads", HEADS)
def test_values_far_apart(ops, heads, dtype, big, small, mode):
    lens = [13, 64, 200] if heads[1] < 10 else [64, 100]
    x = far_apart(heads, lens, dtype, big, small, mode)
    ref = reference(x, lens, x["state"].cpu().numpy(), heads[2] ** -0.5, True)
    o = ops.gated_delta_prefill(*args(x), cu(lens))
    check(o, x["state"], ref, lens, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("mode", ["value then gate", "old state"])
def test_prompt_and_steps_agree(ops, dtype, mode):
    """The same 64 tokens as one prompt and as steps, one token after the other."""
    heads, big, small = (1, 4, 128, 64), 6e4 if dtype is torch.float16 else 1e11, 1e-3 if dtype is torch.float16 else 1.0
    x = far_apart(heads, [64], dtype, big, small, mode)
    y = {**x, "state": x["state"].clone()}
    o = ops.gated_delta_prefill(*args(x), cu([64]))
    steps = torch.cat([ops.gated_delta_step(*[t[i:i + 1] if j < 5 else t for j, t in enumerate(args(y))]) for i in range(64)])
    # each is within the tolerance of the other tests of the exact one
    tol = 2 * 24 * np.sqrt(64) * 2.0 ** -24
    assert ((x["state"] - y["state"]).norm(dim=(-1, -2)) <= tol * y["state"].norm(dim=(-1, -2))).all()
    last = slice(40, 64)
    d = (o[last].float() - steps[last].float()).abs()
    assert (d <= torch.finfo(dtype).eps * steps[last].float().abs() + 12 * tol * steps[last].float().abs().max()).all()


def test_a_range_in_one_sequence_stays_there(ops):
    """Sequences and heads beside one whose values lie far apart keep the bits that they have alone."""
    heads, lens = (1, 4, 128, 64), [100, 100]
    x = make(heads, 200, 2, torch.float16, 3)
    y = {n: t.clone() for n, t in x.items()}
    plain = ops.gated_delta_prefill(*args(x), cu(lens))
    y["v"][110:, 2, 20:36] *= 1e-3
    y["v"][110, 2, 20:36] = 6e4
    y["a"][111, 2] = FORGET
    got = ops.gated_delta_prefill(*args(y), cu(lens))
    assert torch.equal(got[:100], plain[:100]) and torch.equal(x["state"][0], y["state"][0])
    keep = [0, 1, 3]
    assert torch.equal(got[:, keep], plain[:, keep]) and torch.equal(x["state"][1, keep], y["state"][1, keep])


@pytest.mark.parametrize("mode", ["value then gate", "small before big", "old state"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_distance(ops, dtype, mode):
    """Values all of one size and others 2^4 to 2^37 (fp16: to 2^24) of it, a sequence for each distance: around the place where
    pairs stop being enough nothing is lost either."""
    heads = (1, 2, 128, 32)
    distances = range(4, 25 if dtype is torch.float16 else 38)
    lens = [64] * len(distances)
    x = far_apart(heads, lens, torch.float32, 1.0, 1.0, mode, 7)
    x["v"] = torch.where(x["v"] < 0, -1.0, 1.0)
    small = 2.0 ** -10 if dtype is torch.float16 else 1.0
    x["v"] *= small
    x["state"] *= small
    for i, e in enumerate(distances):
        big = 2.0 ** e
        if mode == "value then gate":
            x["v"][64 * i + 10] *= big
        elif mode == "small before big":
            x["v"][64 * i + 35] *= big
        else:
            x["state"][i] *= big
    x = {name: t.to(dtype) if name in "qkvab" else t for name, t in x.items()}
    ref = reference(x, lens, x["state"].cpu().numpy(), 0.125, True)
    o = ops.gated_delta_prefill(*args(x), cu(lens), scale=0.125)
    check(o, x["state"], ref, lens, dtype)


@pytest.mark.parametrize("size", [10.0, 100.0, 1000.0, 5000.0])
@pytest.mark.parametrize("odd", [0.0, 1e-4, 1e-7], ids=["zero", "small", "tiny"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(1, 2, 128, 32), (2, 40, 128, 128)])
def test_keys_far_apart(ops, heads, dtype, odd, size):
    """Large keys, scaled to unit length by the op, with a few beside them that are zero or next to nothing."""
    lens = [64, 100, 20]
    x = make(heads, sum(lens), len(lens), torch.float32, 5)
    x["k"] *= size
    x["k"][5::23] *= odd
    x["q"][3::31] *= odd
    x = {name: t.to(dtype) if name in "qkvab" else t for name, t in x.items()}
    ref = reference(x, lens, x["state"].cpu().numpy(), 0.25, True)
    o = ops.gated_delta_prefill(*args(x), cu(lens), scale=0.25)
    check(o, x["state"], ref, lens, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(1, 2, 128, 32), (2, 40, 128, 128)])
def test_small_betas_after_a_gate(ops, heads, dtype):
    """A gate that forgets everything, tokens of value 0, then one whose beta is next to nothing: its part is all that o has."""
    lens = [64, 90]
    x = make(heads, sum(lens), len(lens), dtype, 9)
    x["a"][:] = -8.0
    for at in (0, 64):
        x["a"][at + 20] = FORGET
        x["v"][at + 20:at + 26] = 0
        x["b"][at + 26:at + 30] = -12.0 if dtype is torch.float16 else -30.0
        x["v"][at + 5] *= 100
    ref = reference(x, lens, x["state"].cpu().numpy(), 0.25, True)
    o = ops.gated_delta_prefill(*args(x), cu(lens), scale=0.25)
    check(o, x["state"], ref, lens, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("norm", [True, False])
def test_keys_that_hold_nothing(ops, norm, dtype):
    """A gate leaves e^-25 of the state; its token's key is zero, or next to it, so that the state does not hold its value, and the
    values after it are zero: what is left of the old state is all there is."""
    heads, lens = (1, 4, 128, 32), [64, 90]
    x = make(heads, sum(lens), len(lens), dtype, 13, norm)
    x["A_log"].zero_()
    x["dt_bias"].fill_(-4.0)
    x["a"][:] = -8.0
    for at in (0, 64):
        x["a"][at + 20] = 29.0
        x["k"][at + 20] *= 0 if norm else 2.0 ** -14
        x["v"][at + 21:at + 40] = 0
    ref = reference(x, lens, x["state"].cpu().numpy(), 0.25, norm)
    o = ops.gated_delta_prefill(*args(x), cu(lens), scale=0.25, qk_norm=norm)
    check(o, x["state"], ref, lens, dtype)


@pytest.mark.parametrize("lens", [[5], [64, 70], [1, 1, 1]], ids=["loop", "chunks", "steps"])
def test_keys_and_queries_past_fp32s_squares(ops, lens):
    """bf16 keys and queries whose squares overflow fp32 count as zero where they are scaled to unit length, also where both do."""
    heads, dtype = (1, 2, 128, 32), torch.bfloat16
    x = make(heads, sum(lens), len(lens), dtype, 3)
    y = {n: t.clone() for n, t in x.items()}
    for name, at in (("k", slice(0, None, 3)), ("q", slice(0, None, 2))):
        x[name][at] = 3e25 * torch.sign(x[name][at] - 0.1)
        y[name][at] = 0
    run = (lambda z: ops.gated_delta_step(*args(z))) if len(lens) == 3 else (lambda z: ops.gated_delta_prefill(*args(z), cu(lens)))
    got, want = run(x), run(y)
    assert torch.isfinite(want).all() and torch.equal(got, want) and torch.equal(x["state"], y["state"])
