"""The committed counter and trace figures of the hot path belong to the sources that are here: bench.py leaves them out of its
line when a fingerprint differs."""
import json
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_profile_of_the_hot_path_fits_its_sources():
    sys.path.insert(0, ROOT)
    import bench
    with open(os.path.join(ROOT, bench.TRAFFIC_FILE)) as f:
        taken_from = json.load(f)["source_sha16"]
    csrc = os.path.join(ROOT, "commbench_amd", "csrc")
    now = {name: bench.source_fingerprint(os.path.join(csrc, name)) for name in taken_from}
    assert now == taken_from, "hot-path sources changed since profiles/hbm_traffic.json was taken: profile them again"
    record = bench.profiled_record("target")
    for name in ("ep_layout_fused_kernel", "ep_permute_tiles_kernel", "ep_combine_staged_kernel"):
        assert record["traffic"][name] > 0 and record["profiled_us"][name] > 0


def test_operators_around_the_hot_path_stay_out_of_its_sources():
    """Their declarations and C entries have files of their own, so that work on them leaves the hot path's figures standing."""
    csrc = os.path.join(ROOT, "commbench_amd", "csrc")
    for name in ("ep_device.h", "ep_abi.hip", "ep_layout.hip", "ep_permute.hip", "ep_combine.hip"):
        with open(os.path.join(csrc, name)) as f:
            text = f.read()
        for word in ("quantize", "grouped_matmul", "few_tokens", "ExpertMatmul"):
            assert word not in text, (name, word)
