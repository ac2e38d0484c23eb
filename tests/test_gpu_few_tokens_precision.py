"""GPU tests of how exact moe_few_tokens is: the error's root mean square beside that of the result's own rounding, and whole
numbers that are right to the bit only if the activation's second term and the fp32 products of the routes arrive.
test_expert_precision.py shows on the CPU that forms without them fail."""
import numpy as np
import pytest
import torch

from commbench_amd import ops

from . import expert_precision as xp
from . import expert_rules as rules
from . import expert_util as xu
from . import precision_cases as cases

pytestmark = pytest.mark.gpu


def run(p, gates, quantised):
    weights = []
    for name in ("w13", "w2"):
        codes = torch.from_numpy(p[name].codes).to(xu.DEV)
        weights.append(codes if quantised else codes.to(torch.bfloat16))
    scales = (None, None)
    if quantised:
        scales = [torch.ones(w.shape[:2], device=xu.DEV) if p.get(s) is None else xu.to_gpu(p[s].astype(np.float32))
                  for w, s in zip(weights, ("s13", "s2"))]
    return xu.f64(ops.moe_few_tokens(xu.bf16_round(p["x"]).to(xu.DEV), xu.to_gpu(p["ids"]), gates, *weights, *scales))


def test_every_kernel_is_among_the_shapes():
    for shapes in (cases.RANDOM, cases.EXACT):
        taken = {rules.few_tokens_kernels(*shape, rules.compute_units()) for shape in shapes}
        assert taken >= {("few", "few"), ("many", "many"), ("tiles", "few"), ("tiles", "tiles")}


@pytest.mark.parametrize("shape", cases.RANDOM, ids=str)
@pytest.mark.parametrize("quantised", [True, False])
def test_error_is_that_of_the_last_rounding(shape, quantised):
    print(f"shape {shape} int8 {quantised}", flush=True)
    p = cases.random_problem(shape, quantised)
    want = xp.layer(p["x"], p["ids"], p["gates"], p["w13"], p["w2"], p["s13"], p["s2"])
    share = xp.error_share(run(p, xu.to_gpu(p["gates"]), quantised), want)
    print(f"share {share:.4f}", flush=True)
    assert share < xp.LIMIT


@pytest.mark.parametrize("shape", cases.EXACT, ids=str)
@pytest.mark.parametrize("quantised", [True, False])
def test_whole_numbers_to_the_bit(shape, quantised):
    print(f"shape {shape} int8 {quantised}", flush=True)
    p = cases.exact_problem(shape)
    np.testing.assert_array_equal(run(p, None, quantised), cases.exact_result(p))
