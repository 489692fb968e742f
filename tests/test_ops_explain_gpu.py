"""A refused argument is named, whichever of its rules it breaks."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from dfssm_b200 import ops
    return ops


def test_rows_more_than_2_to_31_elements_apart(ops):
    mk = lambda *s, t=torch.float16: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    x = dict(q=mk(2, 1, 128), k=mk(2, 1, 128), v=mk(2, 2, 64), a=mk(2, 2), b=mk(2, 2), A_log=mk(2, t=torch.float32),
             dt_bias=mk(2, t=torch.float32), state=mk(2, 2, 64, 128, t=torch.float32))
    far = torch.empty(2 ** 31 + 256, dtype=torch.float16, device="cuda")
    apart = lambda t: far.as_strided(t.shape, (2 ** 31, *t.stride()[1:]))  # noqa: E731
    cu, ws = torch.tensor([0, 2], dtype=torch.int32, device="cuda"), torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    for name in "qkvab":
        with pytest.raises(ValueError, match=f"^{name} must be"):
            ops.gated_delta_step(*{**x, name: apart(x[name])}.values())
        with pytest.raises(ValueError, match=f"^{name} must be"):
            ops.gated_delta_prefill(*{**x, name: apart(x[name])}.values(), cu, workspace=ws)
    with pytest.raises(ValueError, match="^out must be"):
        ops.gated_delta_step(*x.values(), out=apart(x["v"]))
    lg = far.as_strided((2, 50), (2 ** 31, 1)).zero_()  # logits may be as far apart as they like
    u = torch.tensor([0.3, 0.6], device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(ops.sample_filtered(lg, u), ops.sample_filtered(lg.contiguous(), u)))


def test_outputs_of_sampling_that_are_no_triple(ops):
    lg, u = torch.randn(3, 50, device="cuda"), torch.rand(3, device="cuda")
    good = ops.sample_filtered(lg, u)
    for bad in (good[0], good[:2], (*good, good[2]), 5, (1, 2, 3), (good[0], good[1], None)):
        with pytest.raises(ValueError, match="out"):
            ops.sample_filtered(lg, u, out=bad)
    assert torch.equal(ops.sample_filtered(lg, u, out=list(good))[0], good[0])
