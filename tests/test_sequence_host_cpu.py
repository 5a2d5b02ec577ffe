"""The host side of the scan, the linear cross-entropy and AdamW (plans, workspace layouts, launches) under AddressSanitizer and
UndefinedBehaviorSanitizer, with launches written down instead of made (tests/sequence_host_check.cpp)."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "video-classification_amd", "csrc")


def test_host_code_of_the_sequence_operators_under_sanitizers():
    if shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("needs make and hipcc")
    r = subprocess.run(["make", "-C", CSRC, "-j8", "sequencecheck"], capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:verify_asan_link_order=0", UBSAN_OPTIONS="print_stacktrace=1")
    r = subprocess.run([os.path.join(CSRC, "build_asan", "sequence_host_check")], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    assert "ERROR: AddressSanitizer" not in r.stderr and "runtime error" not in r.stderr, r.stderr[-3000:]
    assert r.stdout.startswith("calls ") and int(r.stdout.split()[1].rstrip(",")) > 3000
