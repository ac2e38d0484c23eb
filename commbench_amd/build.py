"""Builds libmi_ep.so (the gfx950 HIP kernels behind the C ABI) in-tree with hipcc."""
import os
import subprocess

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC_DIR = os.path.join(PKG_DIR, "csrc")
LIB_PATH = os.path.join(PKG_DIR, "libmi_ep.so")
SOURCES = ["ep_abi.hip", "ep_host.hip", "ep_layout.hip", "ep_permute.hip", "ep_combine.hip", "ep_expert_abi.hip",
           "ep_quantize.hip", "ep_expert_matmul.hip", "ep_few_tokens.hip"]

# Packed fp32 instructions are switched off for every device compile of this tree.
HIPCC_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-shared", "-Wall", "-Wextra",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def build_library(verbose: bool = False) -> str:
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    cmd = [hipcc, *HIPCC_FLAGS, "-o", LIB_PATH] + [os.path.join(CSRC_DIR, s) for s in SOURCES]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("hipcc failed:\n" + proc.stdout + proc.stderr)
    if verbose:
        print(proc.stderr)
    return LIB_PATH


if __name__ == "__main__":
    print(build_library(verbose=True))
