"""GPU tests of rms_norm_quantize, quantize_rows and dequantize_rows.

Without the norm everything is pinned to the bit: scale and quotient are single fp32 divisions.  With it, a
norm's value y carries at most NORM roundings relative to itself: h = x + r (1), the sum of squares (at most
32 columns of a thread in a row, 6 levels in the wave, 16 waves: 54, halved by the root), division by the
width, adding eps, root, reciprocal (4, the root halving two of them), two products (2): 36."""
import numpy as np
import pytest
import torch

from commbench_amd import _lib, ops
from commbench_amd import workloads as wl

from . import expert_util as xu
from . import gpu_util as gu

pytestmark = pytest.mark.gpu

NORM = 36 * xu.U
E4M3 = 2.0 ** -4


def rows_of(rng, rows, width, spread=1.0):
    return xu.bf16_round(rng.standard_normal((rows, width)) * np.exp(spread * rng.standard_normal((rows, 1))))


def int8_reference(x: torch.Tensor):
    f = x.to(torch.float32).numpy()
    amax = np.abs(f).max(axis=1, keepdims=True)
    scales = np.where(amax > 0, amax / np.float32(127.0), np.float32(1.0)).astype(np.float32)
    return np.rint(f / scales).astype(np.int8), scales


# width: one vector, one wave's exact share, one more, several vectors a lane, one workgroup a row, the largest
@pytest.mark.parametrize("rows,width", [(1, 8), (3, 512), (5, 520), (4, 1032), (7, 2048), (2, 4096), (9, 4104), (3, 7168),
                                        (2, 8200), (2, 16392), (2, 32768), (1000, 256)])
def test_int8_rows_to_the_bit(rows, width):
    print(f"int8 rows {rows} x {width}", flush=True)
    x = rows_of(np.random.default_rng(rows * 7 + width), rows, width)
    if rows > 2:
        x[1] = 0                                             # a row of zeros: scale 1, codes 0
    want_q, want_s = int8_reference(x)
    q, s = ops.quantize_rows(x.to(xu.DEV))
    np.testing.assert_array_equal(s.cpu().numpy(), want_s)
    np.testing.assert_array_equal(q.cpu().numpy(), want_q)
    back = ops.dequantize_rows(q, s)
    want = xu.bf16_round(want_q.astype(np.float32) * want_s)
    np.testing.assert_array_equal(gu.bf16_bits(back), gu.bf16_bits(want))


@pytest.mark.parametrize("rows,width", [(1, 128), (3, 640), (130, 2048), (5, 4224), (17, 7168), (2, 32768)])
@pytest.mark.parametrize("column_major", [False, True])
def test_e4m3_blocks_are_the_workloads_own_payload(rows, width, column_major):
    print(f"e4m3 rows {rows} x {width} column_major {column_major}", flush=True)
    x = rows_of(np.random.default_rng(rows + width), rows, width)
    x[0, :128] = 0
    want_q, want_s = wl.quantize_fp8_blockwise(x)
    q, s = ops.quantize_rows(x.to(xu.DEV), quant="e4m3", column_major_scales=column_major)
    assert s.stride() == ((1, rows) if column_major else (width // 128, 1)) or rows == 1
    np.testing.assert_array_equal(s.cpu().numpy(), want_s.numpy())
    np.testing.assert_array_equal(q.cpu().view(torch.uint8).numpy(), want_q.view(torch.uint8).numpy())
    back = ops.dequantize_rows(q, s)
    want = xu.bf16_round(want_q.to(torch.float32).numpy().reshape(rows, -1, 128) * want_s.numpy()[:, :, None]).view(rows, width)
    np.testing.assert_array_equal(gu.bf16_bits(back), gu.bf16_bits(want))


@pytest.mark.parametrize("magnitude", [1e-38, 1e-33, 1e-30, 1.0, 1e30, 1e37])
@pytest.mark.parametrize("quant", ["int8", "e4m3"])
def test_extreme_magnitudes_to_the_bit(magnitude, quant):
    """Scales around the ends of the normal range take the divisions instead of the corrected reciprocal."""
    x = xu.bf16_round(np.random.default_rng(3).standard_normal((4, 256)) * magnitude)
    q, s = ops.quantize_rows(x.to(xu.DEV), quant=quant)
    if quant == "int8":
        want_q, want_s = int8_reference(x)
        np.testing.assert_array_equal(q.cpu().numpy(), want_q)
        np.testing.assert_array_equal(s.cpu().numpy(), want_s)
    else:
        want_q, want_s = wl.quantize_fp8_blockwise(x)
        np.testing.assert_array_equal(s.cpu().numpy(), want_s.numpy())
        np.testing.assert_array_equal(q.cpu().view(torch.uint8).numpy(), want_q.view(torch.uint8).numpy())


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("quant", ["int8", "e4m3"])
def test_rows_with_infinities_and_nan_read_back_as_nan(bad, quant):
    x = rows_of(np.random.default_rng(4), 3, 512)
    x[1, 200] = bad
    q, s = ops.quantize_rows(x.to(xu.DEV), quant=quant)
    back = ops.dequantize_rows(q, s).cpu()
    touched = slice(0, 512) if quant == "int8" else slice(128, 256)
    assert torch.isnan(back[1, touched].float()).all()
    clean = torch.ones((3, 512), dtype=torch.bool)
    clean[1, touched] = False
    assert torch.isfinite(back.float()[clean]).all()


@pytest.mark.parametrize("rows,width", [(1, 8), (1, 7168), (33, 256), (6, 2056), (5, 4096), (19, 7168), (3, 12288), (2, 32768)])
@pytest.mark.parametrize("quant", ["int8", "e4m3"])
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm_against_64_bits(rows, width, quant, with_residual):
    if quant == "e4m3" and width % 128:
        width = -(-width // 128) * 128
    print(f"norm {rows} x {width} {quant} residual {with_residual}", flush=True)
    rng = np.random.default_rng(rows * 31 + width)
    x, g = rows_of(rng, rows, width), xu.bf16_round(1.0 + 0.2 * rng.standard_normal(width))
    r = rows_of(rng, rows, width) if with_residual else None
    if rows > 2:
        x[1] = 0
        if with_residual:
            r[1] = 0
    eps = 1e-5
    got = ops.rms_norm_quantize(x.to(xu.DEV), g.to(xu.DEV), eps, residual=None if r is None else r.to(xu.DEV), quant=quant,
                                normed=True)
    q, s, normed = got[0], got[1], got[-1]
    h = xu.f64(x) + (xu.f64(r) if with_residual else 0.0)
    eps64 = float(np.float32(eps))
    y = h / np.sqrt((h * h).mean(axis=1, keepdims=True) + eps64) * xu.f64(g)
    y_err = NORM * np.abs(y)
    xu.check_within(xu.f64(normed), y, y_err + xu.BF16 * (np.abs(y) + y_err) + 2.0 ** -133)
    if with_residual:
        assert len(got) == 4
        want = (x.to(torch.float32) + r.to(torch.float32)).to(torch.bfloat16)
        np.testing.assert_array_equal(gu.bf16_bits(got[2]), gu.bf16_bits(want))
    else:
        assert len(got) == 3
    span = width if quant == "int8" else 128
    blocks = y.reshape(rows, -1, span)
    amax = np.abs(blocks).max(axis=2)
    want_s = np.where(amax > 0, amax / (127.0 if quant == "int8" else 448.0), 1.0)
    xu.check_within(xu.f64(s), want_s, (NORM + 2 * xu.U) * want_s)
    values = xu.f64(q).reshape(blocks.shape) * xu.f64(s)[:, :, None]
    step = 0.5 * want_s[:, :, None] if quant == "int8" else np.maximum(E4M3 * np.abs(blocks), 2.0 ** -10 * want_s[:, :, None])
    # half a step around a quotient that is itself off by the errors of y and of the scale
    xu.check_within(values, blocks, step * (1 + 4 * NORM) + (2 * NORM + 4 * xu.U) * np.abs(blocks))


def test_padded_rows_and_in_place_residual():
    rng = np.random.default_rng(8)
    T, H = 37, 1040
    x, r = rows_of(rng, T, H + 24), rows_of(rng, T, H)
    g = xu.bf16_round(1.0 + 0.1 * rng.standard_normal(H)).to(xu.DEV)
    xs = x.to(xu.DEV)[:, :H]                                 # rows H + 24 apart
    want = ops.rms_norm_quantize(xs.contiguous(), g, residual=r.to(xu.DEV))
    stream = r.to(xu.DEV)
    got = ops.rms_norm_quantize(xs, g, residual=stream, update_residual=True)
    assert got[2].data_ptr() == stream.data_ptr()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    wide = torch.zeros((T, H + 8), dtype=torch.bfloat16, device=xu.DEV)
    wide[:, :H] = r.to(xu.DEV)
    again = ops.rms_norm_quantize(xs, g, residual=wide[:, :H])
    for a, b in zip(want, again):
        assert torch.equal(a, b)
    q, s = ops.quantize_rows(xs)
    q2, s2 = ops.quantize_rows(xs.contiguous())
    assert torch.equal(q, q2) and torch.equal(s, s2)


def test_rows_behind_the_limit_stay_as_they_were():
    rows, H, limit = 40, 512, 13
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    x = rows_of(np.random.default_rng(5), rows, H).to(xu.DEV)
    for count in (limit, 0, -1, rows + 5):
        q = torch.full((rows, H), 0x5A, dtype=torch.int8, device=xu.DEV)
        s = torch.full((rows,), -3.0, device=xu.DEV)
        at = torch.tensor([count], dtype=torch.int32, device=xu.DEV)
        _lib.check(lib.mi_ep_quantize_rows(x.data_ptr(), H, at.data_ptr(), rows, H, 0, q.data_ptr(), s.data_ptr(), 1, 1, stream), "quantize")
        out = torch.full((rows, H), 7.0, dtype=torch.bfloat16, device=xu.DEV)
        _lib.check(lib.mi_ep_dequantize_rows(q.data_ptr(), s.data_ptr(), 1, 1, at.data_ptr(), rows, H, 0, out.data_ptr(), stream), "dequantize")
        n = min(max(count, 0), rows)
        want_q, want_s = ops.quantize_rows(x)
        assert torch.equal(q[:n], want_q[:n]) and torch.equal(s[:n], want_s[:n, 0])
        assert bool((q[n:] == 0x5A).all()) and bool((s[n:] == -3.0).all()) and bool((out[n:] == 7.0).all())
        assert torch.equal(out[:n], ops.dequantize_rows(want_q, want_s)[:n])


def test_no_rows():
    x = torch.empty((0, 256), dtype=torch.bfloat16, device=xu.DEV)
    q, s = ops.quantize_rows(x)
    assert q.shape == (0, 256) and s.shape == (0, 1) and ops.dequantize_rows(q, s).shape == (0, 256)
    got = ops.rms_norm_quantize(x, torch.ones(256, dtype=torch.bfloat16, device=xu.DEV), residual=x)
    assert [t.shape[0] for t in got] == [0, 0, 0]


def test_more_rows_than_one_launch_takes():
    """70 million rows: more threads than a launch has."""
    rows = 70_000_000
    free, _ = torch.cuda.mem_get_info()
    if free < 8 << 30:
        pytest.skip("needs 8 GiB of device memory")
    x = torch.zeros((rows, 8), dtype=torch.bfloat16, device=xu.DEV)
    at = torch.tensor([0, 1, (1 << 25) - 1, 1 << 25, (1 << 26) - 1, 1 << 26, rows - 1], device=xu.DEV)
    x[at] = rows_of(np.random.default_rng(2), 7, 8).to(xu.DEV)
    q, s = ops.quantize_rows(x)
    want_q, want_s = ops.quantize_rows(x[at])
    assert torch.equal(q[at], want_q) and torch.equal(s[at], want_s)
    q[at], s[at] = 0, 1.0
    assert not bool(q.any()) and bool((s == 1.0).all())              # all other rows are rows of zeros


def test_one_row_in_a_thousand_threads_is_the_same_as_among_many():
    """Few rows take other launch shapes than many: the same codes either way."""
    x = rows_of(np.random.default_rng(6), 300, 7168).to(xu.DEV)
    g = torch.ones(7168, dtype=torch.bfloat16, device=xu.DEV)
    for quant in ("int8", "e4m3"):
        q, s = ops.quantize_rows(x, quant=quant)
        for n in (1, 2, 255, 256, 257):
            few_q, few_s = ops.quantize_rows(x[:n], quant=quant)
            assert torch.equal(few_q.view(torch.uint8), q[:n].view(torch.uint8)) and torch.equal(few_s, s[:n])
    assert len(ops.rms_norm_quantize(x[:1], g)) == 2
