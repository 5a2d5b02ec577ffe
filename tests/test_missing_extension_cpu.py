"""Without _tensors.so the package loads, the video path is there, and the operators that need it say so."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import sys
sys.modules["vc3d._tensors"] = None  # an import of it fails
import torch, vc3d
from vc3d import ops
from vc3d.capi import Vc3dError
from vc3d.optim import AdamW
from models.model import create_model
from helpers import make_config
create_model(make_config(18, 5), True)
t, y = torch.zeros(2, 3, 8), torch.zeros(2, dtype=torch.int64)
calls = [lambda: vc3d.gated_scan(t), lambda: vc3d.gated_scan_step(t[0], t[0]), lambda: vc3d.linear_cross_entropy(t[0], t[0], y),
         lambda: ops.adamw_step([t], [t], [t], [t], lr=1, beta1=0, beta2=0, eps=0, weight_decay=0, step=1)]
for call in calls:
    try:
        call()
    except Vc3dError as e:
        assert "_tensors.so" in str(e) and "make -C" in str(e), e
    else:
        raise SystemExit("not refused")
print("as it should be")
"""


def test_the_package_loads_without_the_torch_extension():
    pkg = os.path.join(ROOT, "video-classification_amd")
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([pkg, os.path.join(pkg, "lib"), os.path.join(ROOT, "tests"), ROOT]))
    r = subprocess.run([sys.executable, "-c", PROGRAM], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "as it should be" in r.stdout, r.stdout[-1000:] + r.stderr[-2000:]
