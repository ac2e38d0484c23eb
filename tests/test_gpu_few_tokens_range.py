"""GPU tests of moe_few_tokens with activations at the upper end of the range."""
import numpy as np
import pytest
import torch

from commbench_amd import ops

from . import expert_util as xu

pytestmark = pytest.mark.gpu

# tokens, experts, slots, hidden, intermediate: one launch shape for each of the layer's kernels
SHAPES = [(3, 8, 2, 160, 48), (40, 2, 2, 96, 32), (128, 1024, 8, 144, 48), (128, 1024, 8, 528, 144)]


@pytest.mark.parametrize("T,E,K,H,I", SHAPES)
@pytest.mark.parametrize("quantised", [True, False])
@pytest.mark.parametrize("sign", [1, -1])
def test_activations_between_the_largest_bf16_and_the_largest_fp32(T, E, K, H, I, quantised, sign):
    """silu(g) * u = 255/128 * 2^64 * (1 + 3/1024) * 2^63, which is finite in fp32 and rounds to infinity in bf16; the down
    weights bring it back into range.  bf16 weights do so before the sum; int8 codes are summed in fp32 before their
    scale, where two such activations, 2 * 3.396e38, pass fp32's largest value of 3.403e38, so a row of codes has one."""
    print(f"tokens {T} experts {E} slots {K} hidden {H} intermediate {I} int8 {quantised} sign {sign}", flush=True)
    act = 255 / 128 * 2.0 ** 64 * (1 + 3 / 1024) * 2.0 ** 63
    assert np.isfinite(np.float32(act)) and torch.isinf(torch.tensor(act).to(torch.bfloat16))
    rng = np.random.default_rng(T)
    ids, gates = xu.routing(rng, T, E, K)
    x = np.zeros((T, H))
    x[:, 0], x[:, 1] = 1.0, 2.0 ** -10
    w13, w2 = np.zeros((E, 2 * I, H)), rng.integers(-1, 2, (E, H, I)).astype(np.float64)
    gate, up, down = 255 / 128 * 2.0 ** 64, sign * 2.0 ** 63, 2.0 ** -40
    w13[:, :I, 0] = 1.0
    w13[:, I:, 0], w13[:, I:, 1] = 1.0, 3.0
    if quantised:
        w2[:] = 0
        w2[:, np.arange(H), rng.integers(0, I, H)] = rng.choice([-1.0, 1.0], H)
    s13 = np.concatenate([np.full((E, I), gate), np.full((E, I), up)], axis=1).astype(np.float32)
    s2 = np.full((E, H), down, dtype=np.float32)
    bf16 = lambda v: xu.bf16_round(v).to(xu.DEV)
    if quantised:
        weights = (xu.to_gpu(w13.astype(np.int8)), xu.to_gpu(w2.astype(np.int8)), xu.to_gpu(s13), xu.to_gpu(s2))
    else:
        weights = (bf16(w13 * s13[:, :, None].astype(np.float64)), bf16(w2 * down), None, None)
    out = ops.moe_few_tokens(bf16(x), xu.to_gpu(ids), xu.to_gpu(gates), *weights)
    want, bound = xu.few_tokens64(x, ids, gates, w13, w2, s13.astype(np.float64), s2.astype(np.float64))
    xu.check_within(xu.f64(out), want, bound)
