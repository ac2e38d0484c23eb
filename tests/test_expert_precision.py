"""The checks of test_gpu_few_tokens_precision.py on the CPU: a right form passes them, forms that hold the activation or a route's
product in fewer bits do not, on the shapes and inputs of the GPU tests."""
import numpy as np
import pytest

from . import expert_precision as xp
from . import precision_cases as cases


@pytest.mark.parametrize("shape", cases.RANDOM, ids=str)
@pytest.mark.parametrize("quantised", [True, False])
def test_share_of_right_and_wrong_forms(shape, quantised):
    p = cases.random_problem(shape, quantised)
    rows = np.arange(0, shape[0], max(1, shape[0] // 16))       # some tokens are enough to tell them apart
    args = (p["x"][rows], p["ids"][rows], p["gates"][rows], p["w13"], p["w2"], p["s13"], p["s2"])
    want = xp.layer(*args)
    assert xp.error_share(xp.to_bf16(xp.layer(*args, activation_bits=16)), want) < 1.03
    assert xp.error_share(xp.to_bf16(xp.layer(*args, activation_bits=8)), want) > xp.LIMIT
    assert xp.error_share(xp.to_bf16(xp.layer(*args, product_bits=8)), want) > xp.LIMIT


@pytest.mark.parametrize("shape", cases.EXACT, ids=str)
def test_whole_numbers_that_need_the_second_term(shape):
    p = cases.exact_problem(shape)
    want = cases.exact_result(p)
    args = (p["x"], p["ids"], np.ones(p["ids"].shape), p["w13"], p["w2"], None, None)
    rows = np.arange(0, shape[0], max(1, shape[0] // 8))
    some = lambda **bits: xp.to_bf16(xp.layer(p["x"][rows], p["ids"][rows], args[2][rows], p["w13"], p["w2"], None, None, **bits))
    np.testing.assert_array_equal(some(activation_bits=16), want[rows])
    assert (some(activation_bits=8) != want[rows]).any()
    if shape[2] > 1:
        assert (some(product_bits=8) != want[rows]).any()
