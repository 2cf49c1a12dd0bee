"""How libsvsx.so is built: one makefile, which the sources' hash (bench.kernel_src_sha) covers, with one set of flags for the library and for the variants that tools/ builds beside it."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "scalablevectorsearch_amd", "csrc")


def _make(*args):
    return subprocess.run(["make", "-s", "-C", CSRC, *args], capture_output=True, text=True, check=True).stdout


def test_there_is_one_makefile_and_it_builds_every_source():
    makefiles = [f for f in os.listdir(CSRC) if f.lower() in ("makefile", "gnumakefile") or f.endswith(".mk")]
    assert makefiles == ["Makefile"] and not re.search(r"^-?include", open(os.path.join(CSRC, "Makefile")).read(), re.M)
    commands = _make("-n", "-B").splitlines()
    for f in os.listdir(CSRC):
        if f.endswith(".hip"):
            assert sum(f"-c {f} " in c for c in commands) == 1, f
    from bench import kernel_src_sha

    assert '"Makefile"' in open(os.path.join(ROOT, "bench.py")).read() and len(kernel_src_sha()) == 16


def test_no_kernel_has_packed_float32_instructions():
    assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in _make("flags")
    for c in _make("-n", "-B").splitlines():
        if " -c " in c:
            assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in c


@pytest.mark.parametrize("changed", ["Makefile", "svsx_device.h", "../../include/svsx.h"])
def test_objects_follow_what_they_are_made_from(changed):
    """a change to the flags, too, makes every object anew"""
    commands = _make("-n", "-W", changed).splitlines()
    for f in os.listdir(CSRC):
        if f.endswith(".hip"):
            assert any(f"-c {f} " in c for c in commands), f


def test_a_changed_makefile_makes_the_library_stale(monkeypatch):
    from scalablevectorsearch_amd import _lib

    _lib.build()
    calls = []
    monkeypatch.setattr(_lib.subprocess, "check_call", lambda c: calls.append(c))
    real = os.path.getmtime
    monkeypatch.setattr(_lib.os.path, "getmtime", lambda p: real(p) + (1e9 if os.path.basename(p) == "Makefile" else 0))
    _lib.build()
    assert len(calls) == 1


def test_variants_are_built_with_the_flags_of_the_tree():
    tools = os.path.join(ROOT, "tools")
    for f in os.listdir(tools):
        text = open(os.path.join(tools, f), errors="ignore").read() if f.endswith(".sh") else ""
        if "-c svsx_" in text or "svsx_search_$T.hip" in text or "$f.hip" in text:
            assert re.search(r"make -s( -C \S+)? flags", text) and "-ffp-contract" not in text, f
