"""GPU tests of rms_norm_quantize at both ends of the value range: rows whose squares leave fp32, and rows so small that
their scales are subnormal.

NORM as in test_gpu_quantize_rows.py: 36 roundings of a norm's value relative to itself.  A row whose squares overflow or
vanish is summed after a multiplication by a power of two, which rounds nothing but values 2^126 times smaller than the
row's largest; those count in TINY, an absolute bound."""
import numpy as np
import pytest
import torch

from commbench_amd import ops

from . import expert_util as xu
from . import gpu_util as gu

pytestmark = pytest.mark.gpu

NORM = 36 * xu.U
E4M3 = 2.0 ** -4
TINY = 2.0 ** -100


def check_norm(x, r, g, eps, quant):
    """The norm of x (+ r) against 64 bits: codes times scales, scales, and the bf16 rows."""
    rows, width = x.shape
    got = ops.rms_norm_quantize(x.to(xu.DEV), g.to(xu.DEV), eps, residual=None if r is None else r.to(xu.DEV), quant=quant,
                                normed=True)
    q, s, normed = got[0], got[1], got[-1]
    h = xu.f64(x) + (0.0 if r is None else xu.f64(r))
    y = h / np.sqrt((h * h).mean(axis=1, keepdims=True) + float(np.float32(eps))) * xu.f64(g)
    y_err = NORM * np.abs(y) + TINY
    xu.check_within(xu.f64(normed), y, y_err + xu.BF16 * (np.abs(y) + y_err) + 2.0 ** -133)
    span = width if quant == "int8" else 128
    blocks = y.reshape(rows, -1, span)
    amax = np.abs(blocks).max(axis=2)
    want_s = amax / (127.0 if quant == "int8" else 448.0)
    xu.check_within(xu.f64(s), want_s, (NORM + 2 * xu.U) * want_s + TINY)
    values = xu.f64(q).reshape(blocks.shape) * xu.f64(s)[:, :, None]
    step = 0.5 * want_s[:, :, None] if quant == "int8" else np.maximum(E4M3 * np.abs(blocks), 2.0 ** -10 * want_s[:, :, None])
    xu.check_within(values, blocks, step * (1 + 4 * NORM) + (2 * NORM + 4 * xu.U) * np.abs(blocks) + TINY)


# one and more vectors a lane, a wave or a workgroup for a row, few and many rows
SHAPES = [(5, 256), (6, 1024), (4, 2048), (3, 4096), (3, 7168), (260, 7168), (2, 12288), (2, 32768)]


@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("quant", ["int8", "e4m3"])
@pytest.mark.parametrize("with_residual", [False, True])
def test_rows_whose_squares_leave_fp32(rows, width, quant, with_residual):
    """Magnitudes from 1e-39 (subnormal) to 1e37, next to ordinary rows of the same call."""
    print(f"norm range {rows} x {width} {quant} residual {with_residual}", flush=True)
    rng = np.random.default_rng(rows + width)
    for magnitude, eps in ((1e19, 1e-6), (3e25, 1e-5), (1e37, 0.0), (1e-25, 0.0), (1e-38, 0.0), (1e-39, 0.0), (1e-20, 1e-40),
                           (1e-38, 1e-38), (1e-38, 1e-44)):
        x = xu.bf16_round(rng.standard_normal((rows, width)) * magnitude)
        x[rows // 2] = xu.bf16_round(rng.standard_normal(width))
        r = xu.bf16_round(rng.standard_normal((rows, width)) * magnitude) if with_residual else None
        check_norm(x, r, xu.bf16_round(1.0 + 0.2 * rng.standard_normal(width)), eps, quant)


@pytest.mark.parametrize("quant", ["int8", "e4m3"])
def test_one_value_far_above_the_others(quant):
    rng = np.random.default_rng(1)
    for width, big in ((512, 3e38), (4096, 1e30), (7168, 2e22), (32768, 3e38)):
        x = xu.bf16_round(rng.standard_normal((3, width)))
        x[1, 200] = big
        check_norm(x, None, xu.bf16_round(1.0 + 0.2 * rng.standard_normal(width)), 1e-6, quant)


@pytest.mark.parametrize("width", [512, 4096, 7168, 32768])
def test_infinities_and_zeros_stay_what_they_are(width):
    """Rows that really hold an infinity or a NaN read back as NaN, rows of zeros as zeros (as NaN with epsilon 0), next to
    rows of large finite values."""
    rng = np.random.default_rng(2)
    x = xu.bf16_round(rng.standard_normal((5, width)) * 1e25)
    x[0, 3], x[1, 130], x[2] = float("inf"), float("nan"), 0
    g = torch.ones(width, dtype=torch.bfloat16, device=xu.DEV)
    for eps in (1e-6, 0.0):
        q, s = ops.rms_norm_quantize(x.to(xu.DEV), g, eps)
        back = ops.dequantize_rows(q, s).cpu().float()
        assert torch.isnan(back[:2]).all()
        assert torch.isnan(back[2]).all() if eps == 0.0 else not back[2].any()
        assert torch.isfinite(back[3:]).all() and (back[3:].abs().amax(dim=1) > 1).all()


# In units of 2^-149, the least fp32 value: 0 and 1 unit for the scale, quotients far beyond the codes, the last amounts
# where a scale in whole units is coarse.
UNITS = [1, 5, 63, 64, 100, 126, 127, 190, 191, 224, 225, 255, 380, 447, 508, 760, 1016, 3040, 6144, 12160, 16256, 32512, 65280]


@pytest.mark.parametrize("width", [256, 1024, 4096, 7168, 16384])
@pytest.mark.parametrize("quant", ["int8", "e4m3"])
def test_codes_under_subnormal_scales(width, quant):
    """y is a whole number of units to the bit: x = m * 2^-30 and weight 2^-119 under epsilon 1, beside which the mean of the
    squares vanishes.  Scale, quotient and code are then single roundings; a quotient beyond the largest code is
    that code, a scale that rounds to zero is 1."""
    rng = np.random.default_rng(3)
    rows = len(UNITS)
    m = np.zeros((rows, width), dtype=np.float32)
    for i, top in enumerate(UNITS):
        step = max(1, top // 255 + (top % 255 > 0)) if top > 255 else 1
        step = 1 << (step - 1).bit_length()                       # multiples of a power of two: 8 bits of bf16
        m[i] = rng.integers(-(top // step), top // step + 1, width) * step
        m[i, ::128], m[i, 1::128] = top // step * step, -(top // step * step)
    x = torch.from_numpy(m * np.float32(2.0 ** -30)).to(torch.bfloat16)
    assert np.array_equal(x.to(torch.float32).numpy(), m * np.float32(2.0 ** -30))
    assert float((np.float64(m) ** 2).mean(axis=1).max()) * 2.0 ** -60 < 2.0 ** -25       # lost beside epsilon
    g = torch.full((width,), 2.0 ** -119, dtype=torch.bfloat16, device=xu.DEV)
    q, s = ops.rms_norm_quantize(x.to(xu.DEV), g, 1.0, quant=quant)
    y = m * np.float32(2.0 ** -149)
    top = np.float32(127.0 if quant == "int8" else 448.0)
    blocks = y.reshape(rows, -1, width if quant == "int8" else 128)
    scales = (np.abs(blocks).max(axis=2) / top).astype(np.float32)
    scales[scales == 0] = 1.0
    np.testing.assert_array_equal(s.cpu().numpy(), scales)
    quotients = np.clip(blocks / scales[:, :, None], -top, top).astype(np.float32).reshape(rows, width)
    if quant == "int8":
        np.testing.assert_array_equal(q.cpu().numpy(), np.rint(quotients).astype(np.int8))
    else:
        want = torch.from_numpy(quotients).to(torch.float8_e4m3fn)
        np.testing.assert_array_equal(xu.f64(q), xu.f64(want))
    assert gu.bf16_bits(ops.dequantize_rows(q, s)).shape == (rows, width)
