"""What decides whether the native code is built again: objects are remade when the flags change, build() compiles always."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "video-classification_amd", "csrc")


@pytest.mark.parametrize("target", ["all", "hostcheck"])
def test_a_change_of_flags_remakes_every_object(target):
    """make, told that the Makefile is new (-W) and to print only (-n): one compiler line for each HIP source"""
    if shutil.which("make") is None:
        pytest.skip("needs make")
    r = subprocess.run(["make", "-C", CSRC, "-n", "-W", "Makefile", target], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = r.stdout.splitlines()
    for f in os.listdir(CSRC):
        if f.endswith(".hip"):
            assert any(" -c %s " % f in ln for ln in lines), "%s would be left as it is" % f


def test_build_compiles_what_is_built_already(monkeypatch):
    sys.path.insert(0, ROOT)
    try:
        import __graft_entry__ as entry
    finally:
        sys.path.pop(0)
    asked = []
    monkeypatch.setattr(entry.subprocess, "check_call", lambda cmd, **k: asked.append(cmd))
    entry.build()
    native = [cmd for cmd in asked if cmd[0] == "make" and cmd[cmd.index("-C") + 1] == CSRC]
    assert len(native) == 1 and "-B" in native[0]
