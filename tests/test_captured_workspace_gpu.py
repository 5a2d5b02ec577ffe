"""Convs with split-K captured into graphs: each replay gives the eager bits while other calls outgrow the shared workspace and
other graphs, captured on the same stream, run at the same time."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def conv(N, ci, co, seed):
    from vc3d import ops
    from vc3d.capi import lib
    g = torch.Generator().manual_seed(seed)
    d = ops.conv_desc(N, ci, 1, 1, 1, co, 1, 1, 0)
    assert lib.vc_conv3d_workspace_bytes(d, 0) > 0
    x = torch.randn(N, 1, 1, 1, ci, generator=g).bfloat16().cuda()
    w = (torch.randn(co, ci, generator=g) * ci ** -0.5).bfloat16().cuda()
    return lambda: ops.conv3d_fwd(d, x, w)


def test_captured_split_k():
    runs = [conv(64, 2048, 4096, 1), conv(33, 2048, 2048, 2)]
    want = [run().clone() for run in runs]
    torch.cuda.synchronize()
    side, graphs, outs = torch.cuda.Stream(), [], []
    for run in runs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append(run())
    streams = [torch.cuda.Stream() for _ in runs]
    big = conv(64, 4096, 8192, 3)
    for k in range(6):
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        with torch.cuda.stream(side):
            big()  # outgrows what the stream's earlier calls shared
            junk = torch.full((8 << 20,), float("nan"), device="cuda")
        torch.cuda.synchronize()
        del junk
        assert all(torch.equal(o, w) for o, w in zip(outs, want)), k
        assert all(torch.equal(run(), w) for run, w in zip(runs, want)), k
