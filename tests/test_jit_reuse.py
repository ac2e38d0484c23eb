"""What a run-time compilation compiles again for other shapes, and what it does not: a stand-in compiler records its calls."""
import os
import stat

import pytest

from commbench_amd import build as hip_build
from commbench_amd import jit

SHAPED = {"ep_abi.hip", "ep_host.hip", "ep_layout.hip", "ep_permute.hip", "ep_combine.hip"}


@pytest.fixture
def compiler(tmp_path, monkeypatch):
    """A compiler that writes its arguments to a file and one line to its output; returns the sources compiled since the last
    call as {name: arguments}."""
    log, script = tmp_path / "calls", tmp_path / "hipcc"
    script.write_text('#!/bin/sh\nprintf "%s " "$@" | tr -d "\\n" > ' + str(log) + '.$$ && echo >> ' + str(log) + '.$$\n'
                      'while [ $# -gt 0 ]; do if [ "$1" = -o ]; then echo object > "$2"; fi; shift; done\n')
    script.chmod(script.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("HIPCC", str(script))
    jit.init_jit(cache_dir=str(tmp_path / "cache"))

    def compiled():
        found = {}
        for path in tmp_path.glob("calls.*"):
            words = path.read_text().split()
            for word in words:
                if word.endswith(".hip"):
                    assert os.path.basename(word) not in found, "compiled twice"
                    found[os.path.basename(word)] = words
            path.unlink()
        return found
    yield compiled
    jit.init_jit()


def test_other_shapes_compile_the_sources_that_hold_them(compiler):
    first = jit.compile_library(num_topk=2)
    assert set(compiler()) == set(hip_build.SOURCES)
    assert jit.compile_library(num_topk=2) == first and compiler() == {}
    assert jit.compile_library(num_topk=4) != first
    again = compiler()
    assert set(again) == SHAPED
    assert all("-DMI_EP_FIXED_TOPK=4" in words for words in again.values())
    left = [name for name in os.listdir(jit.cache_dir()) if not name.endswith((".so", ".o"))]
    assert left == []                                            # no staging folder, no half-written file


def test_overlaid_sources_are_compiled_with_the_shapes(compiler, tmp_path):
    """An overlay's file may use any fixed shape, also one of a source that holds none as shipped; so may an overlaid header."""
    jit.compile_library(num_topk=2)
    compiler()
    overlay = tmp_path / "overlay"
    overlay.mkdir()
    (overlay / "ep_quantize.hip").write_text("// another\n")
    jit.init_jit(overlay_root=str(overlay), cache_dir=str(tmp_path / "cache"))
    for topk in (2, 4):
        jit.compile_library(num_topk=topk)
        found = compiler()
        assert set(found) == SHAPED | {"ep_quantize.hip"}
        assert f"-DMI_EP_FIXED_TOPK={topk}" in found["ep_quantize.hip"]
    (overlay / "ep_quantize.hip").unlink()
    (overlay / "ep_device.h").write_text("// another\n")
    for topk in (2, 4):
        jit.compile_library(num_topk=topk)
        found = compiler()
        assert set(found) == set(hip_build.SOURCES)
        assert all(f"-DMI_EP_FIXED_TOPK={topk}" in words for words in found.values())


def test_a_failed_compilation_says_why_and_leaves_nothing(compiler, tmp_path, monkeypatch):
    bad = tmp_path / "bad"
    bad.write_text("#!/bin/sh\necho cannot compile >&2\nexit 1\n")
    bad.chmod(bad.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("HIPCC", str(bad))
    with pytest.raises(RuntimeError, match="cannot compile"):
        jit.compile_library(num_topk=2)
    assert os.listdir(jit.cache_dir()) == []
