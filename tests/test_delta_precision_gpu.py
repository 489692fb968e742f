"""How exact the chunked prompt form is on ordinary inputs: 16 half steps of fp32, 16 x 2^-24 of what a head's state has or still
remembers.  Products with operands in pairs are off by 2^-22, four half steps, and three of them follow one another (S k,
T r, u k); a decay has two for its exponent and exp, the sums two; errors of earlier chunks fade with the state or add up in
quadrature, far below the first."""
import numpy as np
import pytest

from test_gated_delta_gpu import args, cu, make, reference

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("decay", [0.0, 0.02, 0.4, 1.6, 6.0])
@pytest.mark.parametrize("heads,lens", [((1, 4, 128, 64), [64, 200, 33]), ((2, 40, 128, 128), [64, 128]), ((3, 3, 64, 48), [100, 64])])
def test_state_of_ordinary_prompts(heads, lens, decay, dtype):
    """Steady decays: at 1.6 a token their sum passes -100 in a chunk, where an fp32 sum would cost 64 half steps."""
    from dfssm_b200 import ops
    x = make(heads, sum(lens), len(lens), dtype, 17)
    x["A_log"].zero_()
    x["dt_bias"].fill_(np.log(np.expm1(decay)) if decay else -40.0)
    x["a"].mul_(0.1)
    ref = reference(x, lens, x["state"].cpu().numpy(), 0.1, True)
    ops.gated_delta_prefill(*args(x), cu(lens), scale=0.1)
    d = np.sqrt(((x["state"].double().cpu().numpy() - ref[1]) ** 2).sum((-1, -2)))
    assert (d <= 16 * 2.0 ** -24 * ref[3]).all(), (d / (2.0 ** -24 * ref[3])).max()
