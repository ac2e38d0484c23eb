"""GPU tests of arguments that the documentation of the expert layer's operators allows, and of their refusals."""
import numpy as np
import pytest
import torch

from commbench_amd import ops

from . import expert_util as xu

pytestmark = pytest.mark.gpu


def test_biases_in_a_list_as_combine_takes_them():
    rng = np.random.default_rng(1)
    T, E, K, H, I = 4, 8, 2, 64, 32
    ids, gates = xu.routing(rng, T, E, K)
    x, b0, b1 = (xu.bf16_round(rng.standard_normal((T, H))).to(xu.DEV) for _ in range(3))
    w13, w2 = (xu.bf16_round(rng.standard_normal(shape) / 8).to(xu.DEV) for shape in ((E, 2 * I, H), (E, H, I)))
    few = lambda bias: ops.moe_few_tokens(x, xu.to_gpu(ids), xu.to_gpu(gates), w13, w2, bias=bias)
    for pair in ((b0, b1), (b0, None), (None, b1), (None, None)):
        assert torch.equal(few(list(pair)), few(pair))
    y, slots = x, torch.arange(T, dtype=torch.int32, device=xu.DEV).view(T, 1)
    assert torch.equal(ops.combine(y, slots, bias=[b0, b1]), ops.combine(y, slots, bias=(b0, b1)))


@pytest.mark.parametrize("eps", [float("nan"), float("inf"), -1e-6, 1e39, 3.5e38])
def test_an_epsilon_that_fp32_cannot_hold_is_refused(eps):
    x = torch.ones((2, 64), dtype=torch.bfloat16, device=xu.DEV)
    with pytest.raises(ValueError, match="eps must be"):
        ops.rms_norm_quantize(x, torch.ones(64, dtype=torch.bfloat16, device=xu.DEV), eps)
