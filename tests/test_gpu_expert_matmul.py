"""GPU tests of grouped_matmul_int8 against 64-bit integers: c is exact, so an output carries the roundings of
int -> fp32, of the product of the two scales and of the product with it (3), and one to bf16."""
import numpy as np
import pytest
import torch

from commbench_amd import _lib, ops

from . import expert_util as xu

pytestmark = pytest.mark.gpu


def segments(counts, align=1):
    padded = -(-np.asarray(counts) // align) * align
    return np.concatenate([[0], np.cumsum(padded)]).astype(np.int32)


def problem(seed, counts, n, k, align=1, extra_rows=0):
    rng = np.random.default_rng(seed)
    off = segments(counts, align)
    rows, E = int(off[-1]) + extra_rows, len(counts)
    return dict(off=off, counts=np.asarray(counts, dtype=np.int32), a=xu.int8_codes(rng, rows, k), b=xu.int8_codes(rng, E, n, k),
                sa=(0.5 + rng.random(rows)).astype(np.float32) / 30, sb=((0.5 + rng.random((E, n))) * k ** -0.5 / 30).astype(np.float32))


def reference(p, silu):
    """(values, bound, rows that belong to an expert)."""
    rows, E = p["a"].shape[0], p["b"].shape[0]
    n = p["b"].shape[1]
    cols = n // 2 if silu else n
    want, bound, mine = np.zeros((rows, cols)), np.zeros((rows, cols)), np.zeros(rows, dtype=bool)
    for e in range(E):
        lo = int(p["off"][e])
        hi = lo + int(p["counts"][e])
        # float64 holds these integer sums exactly (below 2^31)
        c = p["a"][lo:hi].astype(np.float64) @ p["b"][e].astype(np.float64).T
        c *= p["sa"][lo:hi, None].astype(np.float64) * p["sb"][e].astype(np.float64)
        c_err = 3 * xu.U * np.abs(c) * (1 + 1e-6)
        if silu:
            g, u = c[:, :cols], c[:, cols:]
            v = xu.silu64(g) * u
            err = xu.silu_mul_bound(g, u, c_err[:, :cols], c_err[:, cols:])
        else:
            v, err = c, c_err
        want[lo:hi], mine[lo:hi] = v, True
        bound[lo:hi] = err + xu.BF16 * (np.abs(v) + err) + 2.0 ** -133
    return want, bound, mine


def run_raw(p, silu, use_counts=True, rows=None):
    """Through the C ABI on an output of a known pattern."""
    rows = p["a"].shape[0] if rows is None else rows
    E, n, k = p["b"].shape
    cols = n // 2 if silu else n
    out = torch.full((p["a"].shape[0], cols), -77.0, dtype=torch.bfloat16, device=xu.DEV)
    t = {key: xu.to_gpu(p[key]) for key in ("a", "b", "sa", "sb", "off", "counts")}
    _lib.check(_lib.load().mi_ep_grouped_matmul_int8(
        t["a"].data_ptr(), t["sa"].data_ptr(), 1, t["b"].data_ptr(), t["sb"].data_ptr(), t["off"].data_ptr(),
        t["counts"].data_ptr() if use_counts else None, rows, E, n, k, out.data_ptr(), 1 if silu else 0,
        torch.cuda.current_stream().cuda_stream), "matmul")
    torch.cuda.synchronize()
    return out


CASES = [  # counts, out, in: one row; empty experts; odd sizes around every tile edge; few and many rows
    ([1], 8, 16), ([1], 256, 512), ([0, 0, 5, 0], 64, 144), ([3, 0, 17, 1], 40, 80), ([63, 64, 65], 136, 128),
    ([127, 128, 129, 0, 255, 256, 257], 264, 272), ([31, 33, 300], 520, 112), ([16, 15, 9, 1, 2, 0, 7, 8] * 4, 384, 1040),
    ([700], 1032, 2064), ([1] * 100, 48, 64), ([513, 2], 256, 4096), ([40, 50, 60], 2048, 256), ([290, 20], 512, 640)]


@pytest.mark.parametrize("counts,n,k", CASES)
@pytest.mark.parametrize("silu", [False, True])
def test_product_against_integers(counts, n, k, silu):
    if silu:
        n = -(-n // 16) * 16
    print(f"counts {counts[:8]} x {len(counts)} out {n} in {k} silu {silu}", flush=True)
    p = problem(len(counts) * 1000 + n + k, counts, n, k)
    want, bound, _ = reference(p, silu)
    out = ops.grouped_matmul_int8(xu.to_gpu(p["a"]), xu.to_gpu(p["sa"]), xu.to_gpu(p["b"]), xu.to_gpu(p["sb"]),
                                  xu.to_gpu(p["off"]), xu.to_gpu(p["counts"]), activation="silu_mul" if silu else None)
    xu.check_within(xu.f64(out), want, bound)


# 32 experts by four or more column tiles: enough for the large tiles.  Empty, single and full rows around their 32-,
# 64- and 256-row edges; long segments in several tiles.
LARGE = [1, 0, 31, 32, 33, 63, 64, 65, 0, 127, 128, 129, 191, 193, 255, 256, 257, 300, 0, 321, 385, 511, 512, 513, 700, 2, 5, 17,
         0, 40, 90, 1]


@pytest.mark.parametrize("k", [16, 48, 64, 80, 128, 144, 192, 208, 256, 320, 336, 1040])
@pytest.mark.parametrize("n,silu", [(776, False), (1024, False), (1104, True)])
def test_large_tiles_against_integers(n, k, silu):
    """One to many steps over k, whole and partial ones, ragged last columns."""
    print(f"large tiles out {n} in {k} silu {silu}", flush=True)
    p = problem(n + k, LARGE, n, k, extra_rows=70)
    want, bound, mine = reference(p, silu)
    p["sa"][~mine] = np.nan
    out = run_raw(p, silu)
    xu.check_within(xu.f64(out)[mine], want[mine], bound[mine])
    assert bool((out.cpu()[torch.from_numpy(~mine)] == -77.0).all())
    assert torch.equal(run_raw(p, silu), out)                         # and the same again, to the bit


@pytest.mark.parametrize("k", [112, 128, 272, 640])
@pytest.mark.parametrize("n,silu", [(520, False), (1296, True), (896, True)])
def test_tall_tiles_against_integers(n, k, silu):
    """Segments between one and two tiles' rows, the limits on both sides, next to others."""
    counts = [448, 449, 0, 320, 319, 384, 447, 256, 258, 20, 440, 383, 450, 511]
    print(f"tall tiles out {n} in {k} silu {silu}", flush=True)
    p = problem(n + 3 * k, counts, n, k, extra_rows=9)
    want, bound, mine = reference(p, silu)
    p["sa"][~mine] = np.nan
    out = run_raw(p, silu)
    xu.check_within(xu.f64(out)[mine], want[mine], bound[mine])
    assert bool((out.cpu()[torch.from_numpy(~mine)] == -77.0).all())
    assert torch.equal(run_raw(p, silu), out)


@pytest.mark.parametrize("align", [16, 128])
def test_large_tiles_with_pads_strided_scales_and_without_counts(align):
    p = problem(77, LARGE, 768, 272, align)
    want, bound, mine = reference(p, False)
    p["sa"] = np.where(mine, p["sa"], np.nan).astype(np.float32)
    out = run_raw(p, False)
    xu.check_within(xu.f64(out)[mine], want[mine], bound[mine])
    assert bool((out.cpu()[torch.from_numpy(~mine)] == -77.0).all())
    a, b, sb, off, counts = (xu.to_gpu(p[key]) for key in ("a", "b", "sb", "off", "counts"))
    wide = torch.full((p["a"].shape[0], 7), float("nan"), device=xu.DEV)
    wide[:, 3] = xu.to_gpu(p["sa"])
    got = ops.grouped_matmul_int8(a, wide[:, 3:4], b, sb, off, counts)
    rows = torch.from_numpy(mine).to(xu.DEV)
    assert torch.equal(got[rows], out[rows])
    p["sa"] = np.nan_to_num(p["sa"], nan=0.5)
    p["counts"] = np.diff(p["off"]).astype(np.int32)
    want, bound, mine = reference(p, False)
    xu.check_within(xu.f64(run_raw(p, False, use_counts=False))[mine], want[mine], bound[mine])


def test_large_tiles_of_many_experts_and_of_one():
    rng = np.random.default_rng(3)
    for counts, n, k in ((rng.integers(0, 40, 600).tolist(), 512, 64), (rng.integers(5, 30, 1024).tolist(), 264, 48), ([8200], 776, 96)):
        p = problem(len(counts), counts, n, k)
        want, bound, _ = reference(p, False)
        xu.check_within(xu.f64(run_raw(p, False)), want, bound)


def test_large_tiles_on_tables_of_a_layout_that_gave_up():
    """Overlapping, negative and out-of-range segments: in bounds, and an end."""
    p = problem(78, LARGE, 1024, 64)
    rows = p["a"].shape[0]
    rng = np.random.default_rng(1)
    p["off"] = rng.integers(-(1 << 31), 1 << 31, len(LARGE) + 1).astype(np.int32)
    p["counts"] = rng.integers(-(1 << 31), 1 << 31, len(LARGE)).astype(np.int32)
    run_raw(p, False)
    p["off"][:] = 0
    p["counts"][:] = rows                                             # every expert claims every row
    run_raw(p, True)


@pytest.mark.parametrize("silu", [False, True])
def test_extreme_codes(silu):
    """-128 .. 127 at the largest sums, gates far out on both sides."""
    k, n = 8192, 64
    p = problem(5, [70, 3], n, k)
    p["a"][:10], p["b"][0, :20] = -128, -128
    p["a"][10:20], p["b"][0, 20:40] = 127, -128
    p["sa"][:], p["sb"][:] = 1e-4, 1e-2
    want, bound, _ = reference(p, silu)
    xu.check_within(xu.f64(run_raw(p, silu)), want, bound)


@pytest.mark.parametrize("align", [1, 16, 128])
def test_pad_rows_and_rows_behind_stay_as_they_were(align):
    counts = [5, 0, 131, 16, 1]
    p = problem(9, counts, 72, 208, align, extra_rows=11)
    want, bound, mine = reference(p, False)
    p["sa"] = np.where(mine, p["sa"], np.nan).astype(np.float32)       # pads may hold anything
    out = run_raw(p, False)
    xu.check_within(xu.f64(out)[mine], want[mine], bound[mine])
    assert bool((out.cpu()[torch.from_numpy(~mine)] == -77.0).all())
    # without the counts, whole segments are rows
    p["sa"] = np.nan_to_num(p["sa"], nan=0.5)
    p["counts"] = np.diff(p["off"]).astype(np.int32)
    want, bound, mine = reference(p, False)
    out = run_raw(p, False, use_counts=False)
    xu.check_within(xu.f64(out)[mine], want[mine], bound[mine])
    assert bool((out.cpu()[torch.from_numpy(~mine)] == -77.0).all())


def test_segments_are_clamped_to_the_capacity():
    p = problem(10, [40, 100, 60], 64, 64)
    want, bound, _ = reference(p, False)
    out = run_raw(p, False, rows=90)                                   # as if the buffer ended inside expert 1
    xu.check_within(xu.f64(out)[:90], want[:90], bound[:90])
    assert bool((out[90:] == -77.0).all())
    p["off"] = np.array([-5, 20, 2000000000, 2147483647], dtype=np.int32)   # tables of a layout that gave up
    p["counts"] = np.array([-7, 1 << 30, 1 << 30], dtype=np.int32)
    run_raw(p, False)


def test_one_expert_without_tables_and_strided_scales():
    p = problem(11, [77], 120, 336)
    want, bound, _ = reference(p, False)
    a, b, sb = xu.to_gpu(p["a"]), xu.to_gpu(p["b"]), xu.to_gpu(p["sb"])
    plain = ops.grouped_matmul_int8(a, xu.to_gpu(p["sa"]), b, sb)
    xu.check_within(xu.f64(plain), want, bound)
    wide = torch.zeros((77, 5), device=xu.DEV)
    wide[:, 2] = xu.to_gpu(p["sa"])
    assert torch.equal(ops.grouped_matmul_int8(a, wide[:, 2:3], b, sb), plain)
    assert torch.equal(ops.grouped_matmul_int8(a, wide[:, 2], b, sb), plain)
    none = ops.grouped_matmul_int8(a[:0], xu.to_gpu(p["sa"])[:0], b, sb)
    assert none.shape == (0, 120)


def test_weights_beyond_four_gigabytes():
    """Offsets of the last expert's weights pass 32 bits."""
    E, n, k = 5, 8192, 114688
    free, _ = torch.cuda.mem_get_info()
    if free < 8 << 30:
        pytest.skip("needs 8 GiB of device memory")
    rng = np.random.default_rng(1)
    last = xu.int8_codes(rng, n // 256, k)
    b = torch.zeros((E, n, k), dtype=torch.int8, device=xu.DEV)
    at = np.arange(n // 256) * 256 + 255                               # rows spread over the last expert
    b[E - 1, torch.from_numpy(at).to(xu.DEV)] = xu.to_gpu(last)
    a = xu.int8_codes(rng, 3, k)
    off = torch.tensor([0, 0, 0, 0, 0, 3], dtype=torch.int32, device=xu.DEV)
    ones = torch.ones(3, device=xu.DEV)
    sb = torch.full((E, n), 2.0 ** -20, device=xu.DEV)
    out = xu.f64(ops.grouped_matmul_int8(xu.to_gpu(a), ones, b, sb, off))
    want = a.astype(np.float64) @ last.astype(np.float64).T * 2.0 ** -20
    xu.check_within(out[:, at], want, np.abs(want) * (xu.BF16 + 4 * xu.U))
    out[:, at] = 0
    assert not out.any()


def test_replays_of_a_captured_call_follow_the_tables():
    p = problem(12, [50, 0, 200, 6], 192, 384, extra_rows=40)
    a, b, sa, sb = (xu.to_gpu(p[key]) for key in ("a", "b", "sa", "sb"))
    off, counts = xu.to_gpu(p["off"]), xu.to_gpu(p["counts"])
    call = lambda: ops.grouped_matmul_int8(a, sa, b, sb, off, counts, activation="silu_mul")
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for new in ([10, 80, 3, 90], [0, 0, 0, 1], [256, 0, 40, 0]):
        counts.copy_(xu.to_gpu(np.asarray(new, dtype=np.int32)))
        off.copy_(xu.to_gpu(segments(new)))
        total = sum(new)
        eager = call()[:total].clone()
        held.fill_(3.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held[:total], eager)
        assert bool((held[total:] == 3.0).all())


def test_other_stream_gives_the_same():
    p = problem(13, [100, 30], 256, 512)
    a, b, sa, sb, off = (xu.to_gpu(p[key]) for key in ("a", "b", "sa", "sb", "off"))
    want = ops.grouped_matmul_int8(a, sa, b, sb, off)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.grouped_matmul_int8(a, sa, b, sb, off))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
