"""The LSTM cell's packed operands where calls share them: streams, graphs, weights that change in between."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def cell_of(F, H, seed):
    from models.lstm import LSTM
    torch.manual_seed(seed)
    return LSTM(F, H).cuda()


def step(cell, x, h, c):
    from vc3d.lstm import lstm_cell
    p = cell.lstm
    return lstm_cell(x, h, c, p.weight_ih, p.weight_hh, p.bias_ih, p.bias_hh, cell._packed)


def expected(cell, *state):
    """what a module without any history computes"""
    with torch.no_grad():
        out = step(copy.deepcopy(cell), *state)
    torch.cuda.synchronize()
    return out


def equal(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


def test_steps_on_two_streams_after_a_change_of_weights():
    """the first call packs behind 50 ms of other work on its stream; the second, on another stream, may not overtake it"""
    cell, g = cell_of(64, 64, 1), torch.Generator().manual_seed(2)
    args = [tuple(torch.randn(5, 64, generator=g).cuda() for _ in range(3)) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for k in range(3):
        with torch.no_grad():
            cell.lstm.weight_hh.normal_()
        want = [expected(cell, *a) for a in args]
        with torch.no_grad():
            with torch.cuda.stream(streams[k % 2]):
                torch.cuda._sleep(100_000_000)
                first = step(cell, *args[0])
            with torch.cuda.stream(streams[1 - k % 2]):
                second = step(cell, *args[1])
        torch.cuda.synchronize()
        assert equal(first, want[0]) and equal(second, want[1]), k


def test_a_captured_step_follows_the_weights():
    cell, g = cell_of(64, 64, 3), torch.Generator().manual_seed(4)
    args = tuple(torch.randn(5, 64, generator=g).cuda() for _ in range(3))
    expected(cell_of(64, 64, 5), *args)  # (kernels loaded)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        step(cell, *args)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            out = step(cell, *args)
        for k in range(4):
            want = expected(cell, *args)
            graph.replay()
            torch.cuda.synchronize()
            assert equal(out, want), k
            cell.lstm.weight_ih.normal_()
            if k % 2:
                assert equal(step(cell, *args), expected(cell, *args))
