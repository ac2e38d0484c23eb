"""tests/expert_rules.py restates the launchers' rules; when one of these lines changes, the restatement has to follow."""
import os

from commbench_amd import build as hip_build

from . import expert_rules as rules


def source(name):
    with open(os.path.join(hip_build.CSRC_DIR, name)) as f:
        return f.read()


def test_rules_are_the_launchers():
    product = source("ep_expert_matmul.hip")
    for line in ("const bool big = a.num_rows > 12LL * a.num_experts && big_tiles >= 96;",
                 "const long long big_columns = a.silu_mul ? kBigN / 2 : kBigN;",
                 "const long long by_rows = a.num_rows / (kMaxBlocks * kBlockRows);",
                 "const long long by_experts = a.num_rows / 12 < a.num_experts ? a.num_rows / 12 : a.num_experts;",
                 "constexpr int kBigN = 256;", "constexpr int kBlockRows = 64;", "constexpr int kMaxBlocks = 4;",
                 "constexpr int kTallBlocks = 5;"):
        assert line in product, line
    few = source("ep_few_tokens.hip")
    for line in ("const bool many = routes > 8 * a.num_experts;",
                 "return !many && inner > kStageK && items >= static_cast<long long>(items_for_unit) * dev.compute_units;",
                 "tiles(a.hidden, a.intermediate, kSetRows, 4)", "if (tiles(a.intermediate, a.hidden, 2 * kSetRows, 16))",
                 "constexpr int kSetRows = 64, kTileRing = 3;", "if (routes > 2 * a.num_experts) return launch_down<kInt8, 1, 4, 1>"):
        assert line in few, line


def test_rules_on_known_shapes():
    assert rules.product_takes_large_tiles(4694, 14, 1296, True) and not rules.product_takes_large_tiles(4694, 14, 896, True)
    assert not rules.product_takes_large_tiles(4694, 14, 520, False) and rules.product_takes_large_tiles(4694, 14, 1288, False)
    assert rules.few_tokens_kernels(128, 1024, 8, 528, 144) == ("tiles", "tiles")
    assert rules.few_tokens_kernels(128, 1024, 8, 144, 48) == ("tiles", "few")
    assert rules.few_tokens_kernels(1, 256, 8, 7168, 2048) == ("few", "few")
    assert rules.few_tokens_kernels(40, 2, 2, 96, 32) == ("many", "many")
