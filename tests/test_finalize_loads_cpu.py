"""The kernels that read a BatchNorm layer's sums ask for them together: 64 loads of a channel one after the other, each waited for,
made a launch of 5.4 us one of 18.5.  Looked for in the assembly that the build's own command line makes."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "video-classification_amd", "csrc")


def assembly(source, out):
    obj = source.replace(".hip", ".o")
    r = subprocess.run(["make", "-C", CSRC, "-n", "-W", source, obj], capture_output=True, text=True, timeout=120)
    line = next(ln for ln in r.stdout.splitlines() if " -c %s " % source in ln)
    cmd = line.replace(" -c ", " -S --cuda-device-only ").replace("-o " + obj, "-o " + out)
    subprocess.run(cmd.split(), cwd=CSRC, check=True, capture_output=True, timeout=600)
    with open(out) as f:
        return f.read()


def waited_for_alone(code):
    """loads that are issued with none under way and waited for before the next memory instruction"""
    ops = re.findall(r"global_load\w*|buffer_load\w*|s_waitcnt vmcnt\(\d+\)", code)
    return sum("load" in a and b == "s_waitcnt vmcnt(0)" and "load" not in before for before, a, b in zip([""] + ops, ops, ops[1:]))


@pytest.mark.parametrize("source,kernels", [("elementwise.hip", ("18bn_finalize_kernel", "22bn_bwd_finalize_kernel")), ("stem_fwd.hip", ("15stem_fwd_kernel",))])
def test_sums_are_loaded_together(source, kernels, tmp_path):
    if shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("needs make and hipcc")
    text = assembly(source, str(tmp_path / "a.s"))
    for k in kernels:
        code = re.search(r"^(_Z\w*%s\w*):(.*?)\.end_amdhsa_kernel" % k, text, re.S | re.M)[2]
        assert "global_load" in code and waited_for_alone(code) < 24, k
