"""The expert layer's launchers raise a kernel's LDS ceiling on the stream's device, whichever is current (host code, on
stand-ins for the runtime's calls)."""
import os
import re
import subprocess

from commbench_amd import build as hip_build

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
ROCM = os.environ.get("ROCM_HOME", "/opt/rocm")


def test_ceiling_is_raised_on_the_streams_device(tmp_path):
    program = str(tmp_path / "lds_ceiling")
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I" + os.path.join(ROCM, "include"), "-I" + hip_build.CSRC_DIR,
                    "-o", program, os.path.join(CPP, "lds_ceiling.cpp")], check=True, capture_output=True)
    done = subprocess.run([program], capture_output=True, text=True, timeout=30)
    assert done.returncode == 0 and done.stdout == "ok\n", done.stdout


def test_launchers_of_the_expert_layer_use_it():
    for name in ("ep_expert_matmul.hip", "ep_few_tokens.hip"):
        with open(os.path.join(hip_build.CSRC_DIR, name)) as f:
            text = re.sub(r"//.*", "", f.read())
        assert "hipFuncSetAttribute" not in text and "LdsCeiling" in text, name
