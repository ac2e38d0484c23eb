"""GPU tests of rms_norm_quantize on every kernel variant: those of more rows than compute units and of 520 to 1024 columns
among them, in both formats, with and without a residual, against 64 bits as in test_gpu_norm_range.py."""
import numpy as np
import pytest
import torch

from commbench_amd import ops

from . import expert_util as xu
from . import gpu_util as gu
from .test_gpu_norm_range import check_norm

pytestmark = pytest.mark.gpu


# more than 256 rows of 4104 to 8192 columns: four waves a row of four vectors each; up to 256: sixteen of one
@pytest.mark.parametrize("rows,width", [(257, 7168), (300, 4104), (261, 4224), (258, 8192), (256, 7168), (255, 4104), (1100, 5120),
                                        (9, 520), (5, 640), (70, 776), (33, 1024), (1000, 896), (6, 1032), (300, 2304), (259, 12288),
                                        (3, 8200), (5, 16392), (300, 20480)])
@pytest.mark.parametrize("quant", ["int8", "e4m3"])
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm_of_every_shape_against_64_bits(rows, width, quant, with_residual):
    if quant == "e4m3" and width % 128:
        width = -(-width // 128) * 128
    print(f"norm {rows} x {width} {quant} residual {with_residual}", flush=True)
    rng = np.random.default_rng(rows * 5 + width)
    make = lambda: xu.bf16_round(rng.standard_normal((rows, width)) * np.exp(rng.standard_normal((rows, 1))))
    x, r = make(), make() if with_residual else None
    g = xu.bf16_round(1.0 + 0.2 * rng.standard_normal(width))
    check_norm(x, r, g, 1e-5, quant)
    if with_residual:
        stream = ops.rms_norm_quantize(x.to(xu.DEV), g.to(xu.DEV), 1e-5, residual=r.to(xu.DEV), quant=quant)[2]
        want = (x.to(torch.float32) + r.to(torch.float32)).to(torch.bfloat16)
        np.testing.assert_array_equal(gu.bf16_bits(stream), gu.bf16_bits(want))


@pytest.mark.parametrize("quant", ["int8", "e4m3"])
def test_outputs_do_not_depend_on_which_are_asked_for(quant):
    """Codes and scales are the same to the bit with and without bf16(y), in place and not, column-major or not."""
    rng = np.random.default_rng(3)
    for rows, width in ((300, 7168), (20, 7168), (300, 896), (40, 4096)):
        x, r = (xu.bf16_round(rng.standard_normal((rows, width))).to(xu.DEV) for _ in range(2))
        g = xu.bf16_round(1.0 + 0.2 * rng.standard_normal(width)).to(xu.DEV)
        q, s, h = ops.rms_norm_quantize(x, g, residual=r, quant=quant)
        for other in (ops.rms_norm_quantize(x, g, residual=r, quant=quant, normed=True),
                      ops.rms_norm_quantize(x, g, residual=r.clone(), quant=quant, update_residual=True),
                      ops.rms_norm_quantize(x, g, residual=r, quant=quant, column_major_scales=True)):
            assert torch.equal(other[0].view(torch.uint8), q.view(torch.uint8))
            assert torch.equal(other[1], s) and torch.equal(other[2], h)
