"""The pointwise conv kernels keep everything in registers: their loops run with loads to LDS under way, and a register that is spilled
comes back through the same counter (one that was, once, went with wrong results)."""
import os
import re
import shutil

import pytest

from test_finalize_loads_cpu import assembly


def test_pointwise_kernels_spill_nothing(tmp_path):
    if shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("needs make and hipcc")
    text = assembly("pw_conv.hip", str(tmp_path / "a.s"))
    found = re.findall(r"^(_Z\w*pw_kernel\w*):(.*?)\.end_amdhsa_kernel", text, re.S | re.M)
    assert len(found) >= 4
    for name, code in found:
        assert re.search(r"private_segment_fixed_size (\d+)", code)[1] == "0" and "scratch_" not in code, name
