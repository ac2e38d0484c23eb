"""Builds libmi_ep.so (the gfx950 HIP kernels behind the C ABI) in-tree with hipcc."""
import os
import subprocess
import tempfile
from concurrent.futures import ThreadPoolExecutor
from typing import Dict, Sequence

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC_DIR = os.path.join(PKG_DIR, "csrc")
LIB_PATH = os.path.join(PKG_DIR, "libmi_ep.so")
# These hold no shape that may be fixed at build time: one object serves the libraries of all shapes (jit.py).
SHAPE_FREE_SOURCES = ["ep_expert_abi.hip", "ep_quantize.hip", "ep_expert_matmul.hip", "ep_few_tokens.hip"]
SOURCES = ["ep_abi.hip", "ep_host.hip", "ep_layout.hip", "ep_permute.hip", "ep_combine.hip", *SHAPE_FREE_SOURCES]

# Packed fp32 instructions are switched off for every device compile of this tree.
HIPCC_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-shared", "-Wall", "-Wextra",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def _run(cmd: Sequence[str]) -> str:
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("hipcc failed:\n" + proc.stdout + proc.stderr)
    return proc.stderr


def compile_objects(hipcc: str, objects: Dict[str, Sequence[str]]) -> str:
    """Compiles several sources at once: {object file: [source, further flags]}.  Returns what the compiler said."""
    flags = [flag for flag in HIPCC_FLAGS if flag != "-shared"]
    jobs = min(len(objects), int(os.environ.get("MAX_JOBS") or 0) or os.cpu_count() or 1)
    with ThreadPoolExecutor(max(jobs, 1)) as pool:
        said = pool.map(lambda item: _run([hipcc, *flags, *item[1][1:], "-c", "-o", item[0], item[1][0]]), objects.items())
        return "".join(said)


def link_library(hipcc: str, out: str, objects: Sequence[str]) -> str:
    return _run([hipcc, "--offload-arch=gfx950", "-fPIC", "-shared", "-o", out, *objects])


def build_library(verbose: bool = False) -> str:
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    with tempfile.TemporaryDirectory() as folder:
        objects = {os.path.join(folder, name + ".o"): [os.path.join(CSRC_DIR, name)] for name in SOURCES}
        said = compile_objects(hipcc, objects)
        said += link_library(hipcc, LIB_PATH, list(objects))
    if verbose:
        print(said)
    return LIB_PATH


if __name__ == "__main__":
    print(build_library(verbose=True))
