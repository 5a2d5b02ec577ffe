"""What vc_bias_columns refuses before any launch."""
import pytest

PTR = 0x10000  # never read on the host


@pytest.mark.parametrize("bad", [dict(src=None), dict(out=None), dict(rows=0), dict(rows=-1), dict(D=0), dict(D=-4), dict(D=63), dict(D=(1 << 24) + 4)])
def test_the_c_entry_refuses(bad):
    from vc3d import capi
    a = {**dict(src=PTR, out=PTR, rows=4, D=64), **bad}
    assert capi.lib.vc_bias_columns(a["src"], None, a["out"], 1, a["rows"], a["D"], None) == -2
    assert b"bias_columns" in capi.lib.vc_last_error()


def test_there_is_no_cpu_path():
    import torch
    from vc3d import ops
    from vc3d.capi import Vc3dError
    with pytest.raises(Vc3dError):
        ops.bias_columns(torch.zeros(4, 64))
