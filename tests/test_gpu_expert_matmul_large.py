"""GPU tests of grouped_matmul_int8 on shapes that take the large tiles (each says so), against 64-bit integers: tall tiles and
their ragged last columns, capacities that end inside a segment, the largest sums, segments in any order, weights
behind 4 GiB.  Bounds as in test_gpu_expert_matmul.py."""
import numpy as np
import pytest
import torch

from commbench_amd import ops

from . import expert_rules as rules
from . import expert_util as xu
from .test_gpu_expert_matmul import LARGE, problem, reference, run_raw

pytestmark = pytest.mark.gpu

TALL = [448, 449, 0, 320, 319, 384, 447, 256, 258, 20, 440, 383, 450, 511]


def takes_large_tiles(p, silu, rows=None):
    experts, out, _ = p["b"].shape
    assert rules.product_takes_large_tiles(p["a"].shape[0] if rows is None else rows, experts, out, silu)


def check(out, p, silu):
    want, bound, mine = reference(p, silu)
    xu.check_within(xu.f64(out)[mine], want[mine], bound[mine])
    assert bool((out.cpu()[torch.from_numpy(~mine)] == -77.0).all())


# 704 columns: half of the tall tiles' last pair starts where the matrix ends; 648: it starts behind; 1280: a whole number
@pytest.mark.parametrize("k", [112, 128, 272, 640])
@pytest.mark.parametrize("n,silu", [(1408, True), (1296, True), (2560, True), (1288, False), (1536, False)])
def test_segments_of_one_to_two_tiles(n, k, silu):
    print(f"large tiles of {TALL} out {n} in {k} silu {silu}", flush=True)
    p = problem(n + 3 * k, TALL, n, k, extra_rows=9)
    takes_large_tiles(p, silu)
    out = run_raw(p, silu)
    check(out, p, silu)
    assert torch.equal(run_raw(p, silu), out)


@pytest.mark.parametrize("n,silu", [(1408, True), (1288, False)])
@pytest.mark.parametrize("left", [1, 63, 64, 200, 257, 300, 320, 321, 512])
def test_capacity_that_ends_inside_a_segment(n, silu, left):
    """The last expert's 513 rows cut to `left`: another height of tile, and nothing written behind it."""
    counts = LARGE + [513]
    p = problem(left, counts, n, 144)
    rows = int(p["off"][len(LARGE)]) + left
    takes_large_tiles(p, silu, rows)
    out = run_raw(p, silu, rows=rows)
    p["counts"][len(LARGE)] = left
    check(out, p, silu)


@pytest.mark.parametrize("silu", [False, True])
def test_largest_codes(silu):
    """-128 .. 127 at long sums, gates far out on both sides."""
    k, n = 8192, 3584
    p = problem(5, [300, 1100, 640], n, k)
    takes_large_tiles(p, silu)
    p["a"][:100], p["b"][0, :20] = -128, -128
    p["a"][100:200], p["b"][0, 20:40] = 127, -128
    p["sa"][:], p["sb"][:] = 1e-4, 1e-2
    check(run_raw(p, silu), p, silu)


def test_longest_inner_size():
    """131056 columns, the last allowed: codes that are the same along a row, so the sums are known; the largest is 16384 * 131056,
    just below 2^31."""
    rows, n, k = 4100, 1288, 131056
    assert rules.product_takes_large_tiles(rows, 1, n, False) and 16384 * k < 2 ** 31
    rng = np.random.default_rng(6)
    v, c = rng.integers(-128, 128, rows), rng.integers(-128, 128, n)
    v[::7], c[::5] = -128, -128
    spread = lambda code: xu.to_gpu(code.astype(np.int8))[:, None].expand(-1, k).contiguous()
    out = ops.grouped_matmul_int8(spread(v), torch.ones(rows, device=xu.DEV), spread(c)[None], torch.full((1, n), 2.0 ** -20, device=xu.DEV))
    want = np.outer(v, c).astype(np.float64) * k * 2.0 ** -20
    xu.check_within(xu.f64(out), want, np.abs(want) * (xu.BF16 + 4 * xu.U))


@pytest.mark.parametrize("n,silu", [(1408, True), (1288, False)])
def test_segments_in_any_order(n, silu):
    """With the counts given, an expert's rows may lie anywhere: offsets that fall and rise, gaps between."""
    counts = np.asarray(LARGE + [400, 300])
    p = problem(8, counts, n, 208, extra_rows=300)
    rng = np.random.default_rng(9)
    at = 7
    for e in rng.permutation(len(counts)):
        p["off"][e] = at
        at += counts[e] + int(rng.integers(0, 8))
    p["off"][len(counts)] = 0                              # not read: the counts are there
    assert at <= p["a"].shape[0]
    takes_large_tiles(p, silu)
    check(run_raw(p, silu), p, silu)


@pytest.mark.parametrize("silu", [False, True])
def test_weights_behind_4_gib(silu):
    """Three of 80 experts have rows; the last one's weights start behind 10 GiB.  All but a few rows of them are zeros."""
    E, n, k, counts = 80, 4096, 32768, {0: 300, 41: 30, 79: 700}
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GiB of device memory")
    rows = sum(counts.values())
    assert rules.product_takes_large_tiles(rows, E, n, silu) and (E - 1) * n * k > 2 ** 33
    rng = np.random.default_rng(10)
    columns = n // 2 if silu else n
    some = np.sort(rng.choice(columns, 24, replace=False))
    some[-1] = columns - 1
    a, sa = xu.int8_codes(rng, rows, k), (0.5 + rng.random(rows)).astype(np.float32) / 30
    sb = ((0.5 + rng.random((E, n))) * k ** -0.5 / 30).astype(np.float32)
    b = torch.zeros((E, n, k), dtype=torch.int8, device=xu.DEV)
    off = np.zeros(E + 1, dtype=np.int32)
    want, bound, at = np.zeros((rows, columns)), np.full((rows, columns), 2.0 ** -133), 0
    for e in range(E):
        off[e] = at
        if e not in counts:
            continue
        m = slice(at, at + counts[e])
        c = []
        for half in range(2 if silu else 1):
            codes = xu.int8_codes(rng, len(some), k)
            channel = some + half * columns
            b[e, torch.from_numpy(channel).to(xu.DEV)] = xu.to_gpu(codes)
            c.append(a[m].astype(np.float64) @ codes.astype(np.float64).T * sa[m, None].astype(np.float64) * sb[e, channel].astype(np.float64))
        err = [3 * xu.U * np.abs(v) * (1 + 1e-6) for v in c]
        v = xu.silu64(c[0]) * c[1] if silu else c[0]
        v_err = xu.silu_mul_bound(c[0], c[1], err[0], err[1]) if silu else err[0]
        want[m, some], bound[m, some] = v, v_err + xu.BF16 * (np.abs(v) + v_err) + 2.0 ** -133
        at += counts[e]
    off[E] = at
    out = ops.grouped_matmul_int8(xu.to_gpu(a), xu.to_gpu(sa), b, xu.to_gpu(sb), xu.to_gpu(off), activation="silu_mul" if silu else None)
    xu.check_within(xu.f64(out), want, bound)
