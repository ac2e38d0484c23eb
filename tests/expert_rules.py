"""The launchers' choices between kernels, so that a test can say which one its shape takes.  test_expert_rules.py holds
them next to the sources."""
from commbench_amd import ops

COMPUTE_UNITS = 256        # of one MI355X; the GPU tests compare it with what the library reports


def tiles(n, size):
    return -(-n // size)


def product_takes_large_tiles(rows, experts, out, silu):
    columns = out // 2 if silu else out
    by_rows, by_experts = rows // 256, min(rows // 12, experts)
    return rows > 12 * experts and max(by_rows, by_experts) * tiles(columns, 128 if silu else 256) >= 96


def few_tokens_kernels(T, E, K, H, I, compute_units=COMPUTE_UNITS):
    """Which kernels the first and the second product of moe_few_tokens take: "many" (four column blocks), "tiles" or "few"."""
    routes = T * K
    many, met = routes > 8 * E, min(routes, E)
    first = "many" if many else "tiles" if H > 128 and met * tiles(I, 64) >= 4 * compute_units else "few"
    second = "tiles" if not many and I > 128 and met * tiles(H, 128) >= 16 * compute_units else "many" if many else "few"
    return first, second


def compute_units():
    return ops.device_traits()["compute_units"]
